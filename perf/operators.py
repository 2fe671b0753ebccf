"""Cases and plain forms of the operators of rotary and expert encoder layers.

Five operators, each reached through nebw.Device (include/nebw.h has the C
form of each):

  rope          rotary positions on the query and key heads of packed rows
  qk_norm_rope  a norm of each query and key head, then the rotation
  moe_route     the top-k experts of each row, and the rows grouped by expert
  gemm_grouped  one matrix product per expert over ragged groups of rows
  moe_combine   the experts' rows weighted and summed back per row

`own` False computes them in their plain form, True through the framework.
Rows are packed tokens of many sequences; every input is drawn on the GPU
from the seed alone.
"""

import math

import torch

own = False

# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # a query of a few words: rotation only, so the launch is what it costs
        dict(name="rope one short text", op="rope", rows=9, q_heads=12, k_heads=12, head_dim=64,
             rot_dim=64, layout="half", dtype="bf16", packed=True, max_pos=512, theta=1000.0,
             scaling="none", factor=1.0),
        # a whole batch of documents, positions past the trained length, the
        # first half of every head rotated in adjacent pairs
        dict(name="rope document batch", op="rope", rows=65539, q_heads=16, k_heads=16,
             head_dim=64, rot_dim=32, layout="pairs", dtype="bf16", packed=True, max_pos=32768,
             theta=10000.0, scaling="yarn", factor=8.0),
        # fp32 rows of a small model with few key heads, LayerNorm on each head
        dict(name="qk norm fp32 grouped keys", op="qk_norm_rope", rows=4099, q_heads=16, k_heads=4,
             head_dim=96, rot_dim=96, layout="pairs", dtype="f32", packed=False, max_pos=8192,
             theta=10000.0, scaling="ntk", factor=4.0, norm="layer"),
        # a large batch of documents: RMS-normed heads of a packed Q|K|V row
        dict(name="qk norm document batch", op="qk_norm_rope", rows=49999, q_heads=16, k_heads=16,
             head_dim=128, rot_dim=128, layout="half", dtype="bf16", packed=True, max_pos=131072,
             theta=500000.0, scaling="bands", factor=8.0, norm="rms"),
        # the router on one short text, two of eight experts
        dict(name="route one short text", op="moe_route", rows=21, experts=8, top_k=2,
             dtype="f32", score="softmax", renorm=True, dropped=0.0),
        # the router on a batch of documents, eight of many experts
        dict(name="route document batch", op="moe_route", rows=131071, experts=64, top_k=8,
             dtype="bf16", score="softmax", renorm=True, dropped=0.0),
        # the experts' first product for one short text: few rows per expert,
        # so the weights' bytes are the work
        dict(name="grouped one short text", op="gemm_grouped", rows=14, experts=8, top_k=2,
             k=768, n=3840, gated="silu", act="none", gather=True, bias=False, out="bf16",
             skew=0.5),
        # a request of a few texts over many small experts, ragged groups
        dict(name="grouped many experts", op="gemm_grouped", rows=2011, experts=64, top_k=8,
             k=1024, n=1024, gated="silu", act="none", gather=True, bias=False, out="bf16",
             skew=1.0),
        # a batch of documents through the first (gated) product
        dict(name="grouped up batch", op="gemm_grouped", rows=32771, experts=8, top_k=2, k=1024,
             n=8192, gated="gelu_erf", act="none", gather=True, bias=True, out="bf16", skew=0.5),
        # and through the second, whose rows are grouped already
        dict(name="grouped down batch", op="gemm_grouped", rows=32771, experts=8, top_k=2, k=4096,
             n=1024, gated="none", act="none", gather=False, bias=True, out="bf16", skew=0.5),
        # one short text's experts summed
        dict(name="combine one short text", op="moe_combine", rows=17, top_k=2, h=768,
             y_dtype="bf16", out="bf16", residual=False, dropped=0.0),
        # a batch of documents, eight experts a row, added onto the fp32 rows
        dict(name="combine document batch", op="moe_combine", rows=32771, top_k=8, h=1024,
             y_dtype="bf16", out="f32", residual=True, dropped=0.0),
    ]


def _log(rng, lo, hi):
    """A whole number, evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["rope", "qk_norm_rope", "moe_route", "gemm_grouped", "gemm_grouped",
                     "moe_combine"])
    if op in ("rope", "qk_norm_rope"):
        hd = rng.choice([32, 48, 64, 80, 96, 128, 256])
        k_heads = rng.choice([1, 2, 4, 8, 12, 16])
        q_heads = k_heads * rng.choice([1, 1, 2, 4])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        per_row = (q_heads + k_heads) * hd * (2 if dtype == "bf16" else 4)
        rows = _log(rng, 1, max(1, min(100000, 250_000_000 // per_row)))
        rot = rng.choice([hd, hd, hd // 2, hd // 4])
        c = dict(op=op, rows=rows, q_heads=q_heads, k_heads=k_heads, head_dim=hd,
                 rot_dim=max(2, rot - rot % 2), layout=rng.choice(["half", "pairs"]), dtype=dtype,
                 packed=rng.random() < 0.6, max_pos=_log(rng, 64, 131072),
                 theta=rng.choice([1000.0, 10000.0, 160000.0, 1000000.0]),
                 scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                 factor=rng.choice([2.0, 4.0, 8.0]))
        if op == "qk_norm_rope":
            c["norm"] = rng.choice(["rms", "rms", "layer"])
        return c
    if op == "moe_route":
        experts = rng.choice([4, 6, 8, 16, 32, 60, 64, 128, 200, 256])
        return dict(op=op, rows=_log(rng, 1, min(131072, 8_000_000 // experts)), experts=experts,
                    top_k=rng.choice([k for k in (1, 2, 4, 6, 8) if k <= experts]),
                    dtype=rng.choice(["f32", "bf16"]), score=rng.choice(["softmax", "sigmoid"]),
                    renorm=rng.random() < 0.6, dropped=rng.choice([0.0, 0.0, 0.1]))
    if op == "moe_combine":
        h = rng.choice([256, 384, 520, 768, 1024, 1536, 2048])
        k = rng.choice([1, 2, 4, 8])
        return dict(op=op, rows=_log(rng, 1, max(1, 260_000_000 // (h * k))), top_k=k, h=h,
                    y_dtype=rng.choice(["bf16", "bf16", "f32"]), out=rng.choice(["bf16", "f32"]),
                    residual=rng.random() < 0.5, dropped=rng.choice([0.0, 0.0, 0.1]))
    experts = rng.choice([4, 8, 16, 32, 64, 128])
    top_k = rng.choice([1, 2, 4, 8] if experts >= 8 else [1, 2])
    gated = rng.choice(["none", "silu", "gelu_erf"])
    k = rng.choice([256, 384, 512, 768, 1000, 1024, 1536, 2048])
    n = rng.choice([256, 384, 520, 768, 1024, 1536, 2048])
    if gated != "none":
        n = 2 * (n - n % 32)
    out = "f32" if gated == "none" and rng.random() < 0.25 else "bf16"
    act = rng.choice(["none", "gelu_erf"]) if gated == "none" and out == "bf16" else "none"
    rows = _log(rng, 1, max(1, min(65536, 250_000_000_000 // (k * n * top_k))))
    return dict(op=op, rows=rows, experts=experts, top_k=top_k, k=k, n=n, gated=gated, act=act,
                gather=rng.random() < 0.6, bias=rng.random() < 0.5, out=out,
                skew=rng.choice([0.0, 0.5, 1.0, 2.0]))


def work(c):
    op = c["op"]
    if op in ("rope", "qk_norm_rope"):
        e = 2 if c["dtype"] == "bf16" else 4
        n = c["rows"] * (c["q_heads"] + c["k_heads"]) * c["head_dim"]
        table = min(c["rows"], c["max_pos"]) * c["rot_dim"] * 4
        return {"bytes": 2 * n * e + table + 4 * c["rows"],
                "flops": n * (3 if op == "rope" else 7)}
    if op == "moe_route":
        e = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": c["rows"] * (c["experts"] * e + c["top_k"] * 16),
                "flops": c["rows"] * c["experts"] * 4}
    if op == "moe_combine":
        y, o = (2 if c[x] == "bf16" else 4 for x in ("y_dtype", "out"))
        per = c["top_k"] * (c["h"] * y + 8) + c["h"] * (o + (4 if c["residual"] else 0))
        return {"bytes": c["rows"] * per, "flops": 2 * c["rows"] * c["top_k"] * c["h"]}
    m = c["rows"] * c["top_k"]
    n_out = c["n"] if c["gated"] == "none" else c["n"] // 2
    # every row goes somewhere: at most one expert per grouped row is read
    weights = min(c["experts"], m) * c["k"] * c["n"] * 2
    a = (c["rows"] if c["gather"] else m) * c["k"] * 2
    return {"bytes": weights + a + m * n_out * (2 if c["out"] == "bf16" else 4),
            "flops": 2 * m * c["k"] * c["n"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_device = None


def _nebw():
    """The framework's package (it lives beside the header, not on the path)."""
    import sys
    from pathlib import Path

    at = str(Path(__file__).resolve().parent.parent / "npu-embeddings-xdna1_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import nebw

    return nebw


def _dev():
    """One device handle for all cases, on torch's current stream."""
    global _device
    if _device is None:
        _device = _nebw().Device(0, torch_stream=True)
    return _device


class _Staged:
    """A staged weight or table that goes with the state that holds it."""

    def __init__(self, handle):
        self.handle = handle

    def __del__(self):
        try:
            _device.release_weight(self.handle)
        except Exception:
            pass


def _positions(g, rows, max_pos):
    """Positions of the rows of packed sequences of mixed lengths; a few rows
    are single tokens of sequences that go on from anywhere."""
    if rows < 16:
        start = torch.randint(0, max(1, max_pos - rows), (1,), generator=g, device="cuda")
        return (start + torch.arange(rows, device="cuda")).clamp(max=max_pos - 1).int()
    cuts = torch.randint(0, rows, (max(1, rows // 200),), generator=g, device="cuda").sort().values
    at = torch.arange(rows, device="cuda")
    which = torch.searchsorted(cuts, at, right=True)
    starts = torch.cat([cuts.new_zeros(1), cuts])
    offset = torch.randint(0, max(1, max_pos // 2), (starts.numel(),), generator=g, device="cuda")
    return ((at - starts[which] + offset[which]) % max_pos).int()


def _frequencies(c):
    """inv_freq [rot_dim / 2] and the tables' scale, from the formulas (64-bit):
    trained length 4096 (512 below a table of 4096 positions)."""
    n, base, f = c["rot_dim"] // 2, c["theta"], c["factor"]
    trained = 4096 if c["max_pos"] >= 4096 else 512
    i = torch.arange(n, dtype=torch.float64)
    inv = base ** (-i / n)
    if c["scaling"] == "linear":
        return inv / f, 1.0
    if c["scaling"] == "ntk":
        return (base * f ** (n / (n - 1.0)) if n > 1 else base * f) ** (-i / n), 1.0
    if c["scaling"] == "yarn":
        def turn(beta):  # the index whose frequency turns beta times in the trained length
            return n * math.log(trained / (beta * 2 * math.pi)) / math.log(base)
        lo = max(0.0, math.floor(turn(32.0)))
        hi = min(n - 1.0, math.ceil(turn(1.0)))
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    if c["scaling"] == "bands":
        turns = trained * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv * keep + inv / f * (1 - keep), 1.0
    return inv, 1.0


def _routing(c, g):
    """Expert ids [rows, top_k] of a skewed router, and the grouping they give."""
    scores = torch.randn(c["rows"], c["experts"], generator=g, device="cuda")
    scores += c["skew"] * torch.randn(c["experts"], generator=g, device="cuda")
    ids = scores.topk(c["top_k"], dim=1).indices.reshape(-1)
    order = ids.sort(stable=True)
    edges = torch.arange(c["experts"] + 1, device="cuda")
    off = torch.searchsorted(order.values, edges).int()
    return off, (order.indices // c["top_k"]).int()


def _inputs(c, seed):
    """Everything drawn from the seed."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, s = c["op"], {}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if op in ("rope", "qk_norm_rope"):
        t, hd = _TYPES[c["dtype"]], c["head_dim"]
        qw, kw = c["q_heads"] * hd, c["k_heads"] * hd
        # Q|K|V rows of a fused projection, or queries and keys of their own
        x = randn(c["rows"], qw + 2 * kw if c["packed"] else qw + kw).to(t)
        s["q"] = x[:, :qw] if c["packed"] else x[:, :qw].contiguous()
        s["k"] = x[:, qw:qw + kw] if c["packed"] else x[:, qw:].contiguous()
        s["pos"] = _positions(g, c["rows"], c["max_pos"])
        if op == "qk_norm_rope":
            for side in "qk":
                s[side + "_gamma"] = 1 + 0.2 * randn(hd)
                s[side + "_beta"] = 0.2 * randn(hd) if c["norm"] == "layer" else None
    elif op == "moe_route":
        s["logits"] = (1.5 * randn(c["rows"], c["experts"])).to(_TYPES[c["dtype"]])
        if c["dropped"]:  # padding rows: no expert at all
            gone = torch.rand(c["rows"], generator=g, device="cuda") < c["dropped"]
            s["logits"] = torch.where(gone[:, None], -math.inf, s["logits"])
    elif op == "moe_combine":
        m = c["rows"] * c["top_k"]
        s["y"] = randn(m, c["h"]).to(_TYPES[c["y_dtype"]])
        s["row_dst"] = torch.randperm(m, generator=g, device="cuda").int()
        w = torch.rand(c["rows"], c["top_k"], generator=g, device="cuda") + 0.05
        s["weights"] = w / w.sum(1, keepdim=True)
        if c["dropped"]:  # padding rows: they went to no expert
            gone = torch.rand(c["rows"], generator=g, device="cuda") < c["dropped"]
            s["weights"] = torch.where(gone[:, None], 0.0, s["weights"])
            s["row_dst"] = torch.where(gone[:, None], -1, s["row_dst"].view(c["rows"], -1)).int()
        s["residual"] = randn(c["rows"], c["h"]) if c["residual"] else None
    else:
        s["off"], s["src"] = _routing(c, g)
        m = c["rows"] * c["top_k"]
        s["a"] = randn(c["rows"] if c["gather"] else m, c["k"]).to(torch.bfloat16)
        s["w"] = (randn(c["experts"], c["k"], c["n"]) / math.sqrt(c["k"])).to(torch.bfloat16)
        s["bias"] = 0.1 * randn(c["experts"], c["n"]) if c["bias"] else None
    return s


def prepare(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    s["case"], op = c, c["op"]
    if op in ("rope", "qk_norm_rope"):
        inv, scale = _frequencies(c)
        t, qw, kw = _TYPES[c["dtype"]], s["q"].shape[1], s["k"].shape[1]
        s["q_out"] = torch.empty(c["rows"], qw, dtype=t, device="cuda")
        s["k_out"] = torch.empty(c["rows"], kw, dtype=t, device="cuda")
        # the tables that a program keeps for its positions
        angle = torch.arange(c["max_pos"], dtype=torch.float64, device="cuda")[:, None] * inv.cuda()
        s["cos"], s["sin"] = (angle.cos() * scale).float(), (angle.sin() * scale).float()
    elif op == "moe_route":
        m = c["rows"] * c["top_k"]
        s["ids"] = torch.empty(c["rows"], c["top_k"], dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty(c["rows"], c["top_k"], device="cuda")
        s["off"] = torch.empty(c["experts"] + 1, dtype=torch.int32, device="cuda")
        s["src"] = torch.full((m,), -1, dtype=torch.int32, device="cuda")
        s["dst"] = torch.empty(c["rows"], c["top_k"], dtype=torch.int32, device="cuda")
    elif op == "moe_combine":
        s["out"] = torch.empty(c["rows"], c["h"], dtype=_TYPES[c["out"]], device="cuda")
    else:
        n_out = c["n"] if c["gated"] == "none" else c["n"] // 2
        s["out"] = torch.empty(c["rows"] * c["top_k"], n_out, dtype=_TYPES[c["out"]],
                               device="cuda")
        s["sizes"] = s["off"].tolist()
    if own:
        _stage(s, c)
    return s


def _stage(s, c):
    """What a program keeps of the framework's: staged weights and tables, the
    descriptions of its heads, a workspace."""
    nebw, dev, op = _nebw(), _dev(), c["op"]
    if op in ("rope", "qk_norm_rope"):
        inv, scale = _frequencies(c)  # the case's own set
        s["rope"] = _Staged(dev.stage_rope(inv.numpy(), c["max_pos"], scale))
        for side in "qk":
            s[side + "_heads"] = nebw.Heads.of(
                s[side], c[side + "_heads"], out=s[side + "_out"], gamma=s.get(side + "_gamma"),
                beta=s.get(side + "_beta"))
    elif op == "moe_route":
        size = nebw.moe_route_workspace(c["rows"], c["experts"], c["top_k"])
        s["ws"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    elif op == "gemm_grouped":
        s["experts"] = _Staged(dev.stage_experts(s["w"], gated=c["gated"] != "none"))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(s):
    return (_framework if own else _plain)(s, s["case"])


def _framework(s, c):
    nebw, dev, op = _nebw_module(), _device, c["op"]
    if op == "rope":
        dev.rope(s["q_heads"], s["k_heads"], c["rows"], c["head_dim"], s["rope"].handle, s["pos"],
                 layout=_LAYOUTS[c["layout"]])
        return s["q_out"], s["k_out"]
    if op == "qk_norm_rope":
        dev.qk_norm_rope(s["q_heads"], s["k_heads"], c["rows"], c["head_dim"],
                         norm=_NORMS[c["norm"]], eps=1e-6, rope=s["rope"].handle, pos=s["pos"],
                         layout=_LAYOUTS[c["layout"]])
        return s["q_out"], s["k_out"]
    if op == "moe_route":
        dev.moe_route(s["logits"], c["rows"], c["experts"], c["top_k"], s["ids"], s["weights"],
                      s["off"], s["src"], s["dst"], s["ws"], score=_SCORES[c["score"]],
                      renorm=c["renorm"])
        return s["ids"], s["weights"], s["off"], s["src"], s["dst"]
    if op == "moe_combine":
        dev.moe_combine(s["y"], s["row_dst"], s["weights"], c["rows"], c["top_k"], c["h"],
                        s["out"], residual=s["residual"])
        return s["out"]
    gated = c["gated"] != "none"
    act = _GATES[c["gated"]] if gated else _ACTS[c["act"]]
    dev.gemm_grouped(s["experts"].handle, s["a"], s["a"].shape[0], s["off"],
                     c["rows"] * c["top_k"], c["k"], c["n"], s["out"],
                     row_src=s["src"] if c["gather"] else None, bias=s["bias"], act=act,
                     c_dtype=nebw.BF16 if c["out"] == "bf16" else nebw.F32)
    return s["out"]


_LAYOUTS = {"half": 0, "pairs": 1}
_NORMS = {"rms": 1, "layer": 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
_GATES = {"silu": 0, "gelu_erf": 1}
_ACTS = {"none": 0, "gelu_erf": 2}
_module = None


def _nebw_module():
    global _module
    if _module is None:
        _module = _nebw()
    return _module


def _heads_plain(x, heads, gamma, beta, cos, sin, c):
    """The norm and the rotation of one side's heads, in 32 bits."""
    v = x.float().reshape(x.shape[0], heads, c["head_dim"])
    if c["op"] == "qk_norm_rope":
        if c["norm"] == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * gamma
        if beta is not None:
            v = v + beta
    r = c["rot_dim"]
    turned, rest = v[..., :r], v[..., r:]
    if c["layout"] == "half":
        a, b = turned[..., :r // 2], turned[..., r // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1).reshape(x.shape[0], -1).to(x.dtype)


def _gelu(x):
    return 0.5 * x * (1 + torch.erf(x / math.sqrt(2.0)))


def _plain(s, c):
    op = c["op"]
    if op in ("rope", "qk_norm_rope"):
        pos = s["pos"].long()
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        return tuple(_heads_plain(s[x], c[x + "_heads"], s.get(x + "_gamma"), s.get(x + "_beta"),
                                  cos, sin, c) for x in "qk")
    if op == "moe_route":
        return _route_plain(s["logits"].float(), c)
    if op == "moe_combine":
        dst = s["row_dst"].long().reshape(c["rows"], c["top_k"])
        y = torch.where((dst >= 0)[:, :, None], s["y"][dst.clamp(min=0)].float(), 0.0)
        out = (y * s["weights"][:, :, None]).sum(1)
        if s["residual"] is not None:
            out = out + s["residual"]
        return out.to(_TYPES[c["out"]])
    a = s["a"][s["src"].long()] if c["gather"] else s["a"]
    parts, sizes = [], s["sizes"]
    for e in range(c["experts"]):
        if sizes[e + 1] > sizes[e]:
            v = a[sizes[e]:sizes[e + 1]].float() @ s["w"][e].float()
            if s["bias"] is not None:
                v = v + s["bias"][e]
            if c["gated"] != "none":
                up, gate = v.chunk(2, 1)
                v = up * (gate / (1 + torch.exp(-gate)) if c["gated"] == "silu" else _gelu(gate))
            elif c["act"] == "gelu_erf":
                v = _gelu(v)
            parts.append(v.to(_TYPES[c["out"]]))
    return torch.cat(parts)


def _route_plain(x, c):
    """Softmax or sigmoid scores, the top k by logit (ties to the lower
    index), the chosen weights, and the stable grouping by expert.  A logit
    of -inf is never chosen: its place has id -1, weight 0 and no row."""
    e, k = c["experts"], c["top_k"]
    best = x.sort(dim=1, descending=True, stable=True)
    ids, chosen = best.indices[:, :k], best.values[:, :k]
    there = chosen > -math.inf
    if c["score"] == "softmax":
        top = best.values[:, :1].clamp(min=-3e38)
        w = torch.exp(chosen - top)
        total = w if c["renorm"] else torch.exp(x - top)
    else:
        w = total = 1 / (1 + torch.exp(-chosen))
    if c["renorm"] or c["score"] == "softmax":
        w = w / total.sum(1, keepdim=True)
    w = torch.where(there, w, 0.0)
    ids = torch.where(there, ids, -1)
    flat = torch.where(there, ids, e).reshape(-1)
    order = flat.sort(stable=True)
    off = torch.searchsorted(order.values, torch.arange(e + 1, device=x.device)).int()
    src = torch.where(order.values < e, order.indices // k, -1).int()
    place = torch.empty_like(order.indices)
    place[order.indices] = torch.arange(flat.numel(), device=x.device)
    dst = torch.where(flat < e, place, -1).int().reshape(-1, k)
    return ids.int(), w, off, src, dst


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    op = c["op"]
    if op in ("rope", "qk_norm_rope"):
        inv, scale = _frequencies(c)
        # each pair as a complex number, turned by its angle
        turn = torch.polar(torch.full((c["rows"], inv.numel()), scale, dtype=torch.float64,
                                      device="cuda"),
                           s["pos"].double()[:, None] * inv.cuda())
        out, r = [], c["rot_dim"]
        for x in "qk":
            v = s[x].double().view(c["rows"], c[x + "_heads"], c["head_dim"])
            if op == "qk_norm_rope":
                if c["norm"] == "layer":
                    v = (v - v.mean(-1, keepdim=True)) / (v.var(-1, keepdim=True, correction=0)
                                                          + 1e-6).sqrt()
                    v = v * s[x + "_gamma"].double() + s[x + "_beta"].double()
                else:
                    v = v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt()
                    v = v * s[x + "_gamma"].double()
            v = v.clone()
            first = slice(0, r // 2) if c["layout"] == "half" else slice(0, r, 2)
            second = slice(r // 2, r) if c["layout"] == "half" else slice(1, r, 2)
            z = torch.complex(v[..., first], v[..., second]) * turn[:, None]
            v[..., first], v[..., second] = z.real, z.imag
            out.append(v.reshape(c["rows"], -1))
        return tuple(out)
    if op == "moe_route":
        x = s["logits"].double()
        score = torch.softmax(x, 1) if c["score"] == "softmax" else torch.sigmoid(x)
        order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :c["top_k"]]
        w = score.gather(1, order)
        if c["renorm"]:
            w = w / w.sum(1, keepdim=True)
        w = torch.where(x.gather(1, order).isinf(), 0.0, w)
        return None, w, None, None, None
    if op == "moe_combine":
        place = s["row_dst"].long().view(c["rows"], c["top_k"])
        out = torch.zeros(c["rows"], c["h"], dtype=torch.float64, device="cuda")
        for j in range(c["top_k"]):
            there = (place[:, j] >= 0).double() * s["weights"][:, j].double()
            out += there[:, None] * s["y"][place[:, j].clamp(min=0)].double()
        return out if s["residual"] is None else out + s["residual"].double()
    a = s["a"].double()
    if c["gather"]:
        a = a[s["src"].long()]
    edges = s["off"].tolist()
    out = torch.empty(a.shape[0], c["n"], dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(zip(edges, edges[1:])):
        torch.mm(a[lo:hi], s["w"][e].double(), out=out[lo:hi])
        if s["bias"] is not None:
            out[lo:hi] += s["bias"][e].double()
    if c["gated"] != "none":
        f = c["n"] // 2
        gate = out[:, f:]
        phi = torch.sigmoid(gate) if c["gated"] == "silu" else \
            torch.special.ndtr(gate)
        return out[:, :f] * gate * phi
    return out * torch.special.ndtr(out) if c["act"] == "gelu_erf" else out
