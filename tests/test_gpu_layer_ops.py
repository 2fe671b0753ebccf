"""The rotary and expert operators on a B200, through the C ABI, against a
plain computation in 64 bits on the same operands.

Tolerances count roundings: a stored bf16 value is off by at most 2^-8 of
itself (half a step), an fp32 one by 2^-24, and the fp32 arithmetic before it
by the bound stated at each comparison.  Whole numbers are exact.
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24  # fp32 unit roundoff
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def assert_close(got, want, before):
    """|got - want| within the fp32 error `before` plus one rounding to got's type."""
    r = half_step(got.dtype)
    g = got.double()
    tol = before + r * (want.abs() + before) + 1e-37
    bad = ~((g - want).abs() <= tol)
    assert not bad.any(), (
        f"{int(bad.sum())} of {bad.numel()} values off, first at {bad.nonzero()[0].tolist()}: "
        f"{g[bad][0].item()} for {want[bad][0].item()} (tolerance {tol[bad][0].item():.3g})")


# ---------------------------------------------------------------------------
# rotary positions and head norms
# ---------------------------------------------------------------------------

def heads_reference(x, heads, hd, inv, scale, pos, pairs, norm=0, gamma=None, beta=None, eps=0.0):
    """(value, bound of the fp32 error) of one side's heads, in 64 bits."""
    v = x.double().reshape(x.shape[0], heads, hd)
    err = torch.zeros_like(v)
    if norm:
        size = v.abs()
        if norm == 2:
            # the mean's sum is off by hd units of its terms at most
            size = size + size.mean(-1, keepdim=True)
            v = v - v.mean(-1, keepdim=True)
            err = (hd + 2) * U * size
        inv_std = 1.0 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
        # hd fused adds, a divide, a square root, three products; the mean's
        # error reaches the squares as twice its share
        rel = (hd + 8) * U + (err.amax(-1, keepdim=True) * inv_std if norm == 2 else 0.0)
        err = (err * inv_std + v.abs() * inv_std * rel) * gamma.double().abs()
        v = v * inv_std * gamma.double()
        if norm == 2:
            v = v + beta.double()
            err = err + U * v.abs()
    r = 2 * len(inv)
    if r:
        angle = pos.double()[:, None] * torch.tensor(inv, dtype=torch.float64, device="cuda")
        c, s = (angle.cos() * scale)[:, None], (angle.sin() * scale)[:, None]
        a, b = (v[..., 0:r:2], v[..., 1:r:2]) if pairs else (v[..., :r // 2], v[..., r // 2:r])
        ea, eb = (err[..., 0:r:2], err[..., 1:r:2]) if pairs else \
            (err[..., :r // 2], err[..., r // 2:r])
        big = abs(scale)
        # two rounded table entries, a product, a fused add; the sines of the
        # two double evaluations differ by 1e-15 of the angle at most
        turn = (4 * U + 1e-15 * angle.abs()[:, None]) * big * (a.abs() + b.abs()) + big * (ea + eb)
        na, nb = a * c - b * s, b * c + a * s
        out, oerr = v.clone(), err.clone()
        if pairs:
            out[..., 0:r:2], out[..., 1:r:2] = na, nb
            oerr[..., 0:r:2], oerr[..., 1:r:2] = turn, turn
        else:
            out[..., :r // 2], out[..., r // 2:r] = na, nb
            oerr[..., :r // 2], oerr[..., r // 2:r] = turn, turn
        v, err = out, oerr
    return v.reshape(x.shape), err.reshape(x.shape)


HEAD_CASES = [
    # rows, q heads, k heads, head_dim, rot_dim, dtype
    (1, 1, 1, 64, 64, "bf16"),
    (1, 32, 8, 128, 128, "bf16"),
    (3, 12, 12, 32, 32, "bf16"),
    (77, 12, 12, 64, 64, "bf16"),
    (130, 16, 4, 96, 96, "bf16"),     # three vectors of eight pairs a half
    (65, 5, 3, 80, 80, "bf16"),
    (65, 3, 1, 64, 32, "bf16"),       # part of the head
    (65, 3, 1, 64, 16, "bf16"),
    (65, 2, 2, 64, 20, "bf16"),       # no whole vector of pairs
    (33, 2, 1, 64, 2, "bf16"),
    (33, 2, 1, 2, 2, "bf16"),
    (33, 3, 2, 6, 4, "bf16"),
    (19, 2, 2, 256, 256, "bf16"),
    (19, 2, 2, 256, 64, "bf16"),
    (19, 7, 1, 48, 48, "bf16"),
    (5, 2, 1, 250, 130, "bf16"),
    (1, 16, 2, 64, 64, "f32"),
    (77, 12, 12, 64, 64, "f32"),
    (41, 6, 2, 96, 48, "f32"),
    (41, 3, 1, 40, 8, "f32"),
    (41, 3, 1, 38, 6, "f32"),
    (9, 2, 2, 256, 256, "f32"),
    (2100, 4, 2, 64, 64, "bf16"),
]


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("norm", [0, 1, 2])
@pytest.mark.parametrize("rows,qh,kh,hd,rot,dtype", HEAD_CASES)
def test_heads_match_64_bits(device, rows, qh, kh, hd, rot, dtype, norm, pairs):
    import nebw
    t = TYPES[dtype]
    g = gen(rows * 31 + hd * 7 + rot + norm)
    qkv = (2 * torch.randn(rows, (qh + 2 * kh) * hd, generator=g, device="cuda") + 0.3).to(t)
    q, k = qkv[:, :qh * hd], qkv[:, qh * hd:(qh + kh) * hd]
    max_pos = 40000
    pos = torch.randint(0, max_pos, (rows,), generator=g, device="cuda").int()
    pos[0] = max_pos - 1
    inv, scale = nebw.rope_freqs(10000.0, rot, "yarn", factor=4.0, orig_len=4096)
    h = device.stage_rope(inv, max_pos, scale)
    gam = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)]
    bet = [0.5 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)]
    want = [heads_reference(x, n, hd, inv, scale, pos, pairs, norm, gam[i], bet[i], 1e-5)
            for i, (x, n) in enumerate(((q, qh), (k, kh)))]
    before = qkv.clone()

    def call(out_q, out_k):
        hq = nebw.Heads.of(q, qh, out=out_q, gamma=gam[0], beta=bet[0])
        hk = nebw.Heads.of(k, kh, out=out_k, gamma=gam[1], beta=bet[1])
        if norm:
            device.qk_norm_rope(hq, hk, rows, hd, norm=norm, eps=1e-5, rope=h, pos=pos,
                                layout=int(pairs))
        else:
            device.rope(hq, hk, rows, hd, h, pos, layout=int(pairs))

    try:
        # into other rows (of another stride, with a margin that stays)
        out = torch.full((rows, (qh + kh) * hd + 16), 7.0, dtype=t, device="cuda")
        oq, ok = out[:, :qh * hd], out[:, qh * hd:(qh + kh) * hd]
        call(oq, ok)
        device.sync()
        assert torch.equal(qkv, before)
        assert (out[:, (qh + kh) * hd:] == 7.0).all()
        assert_close(oq, *want[0])
        assert_close(ok, *want[1])
        # and in place: the same bits, the values not touched
        call(None, None)
        device.sync()
        assert torch.equal(q, oq) and torch.equal(k, ok)
        assert torch.equal(qkv[:, (qh + kh) * hd:], before[:, (qh + kh) * hd:])
    finally:
        device.release_weight(h)


@pytest.mark.parametrize("shift", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_heads_at_any_alignment_and_stride(device, dtype, shift):
    """Rows that start off a 16-byte boundary, odd row strides: the same bits
    as the aligned call."""
    import nebw
    t, rows, heads, hd = TYPES[dtype], 23, 3, 64
    g = gen(shift)
    x = torch.randn(rows, heads * hd, generator=g, device="cuda").to(t)
    gamma = torch.randn(hd + 1, generator=g, device="cuda")[1:]  # four bytes off too
    pos = torch.arange(rows, device="cuda").int()
    inv, scale = nebw.rope_freqs(10000.0, hd)
    h = device.stage_rope(inv, 64, scale)
    try:
        outs = []
        for pad in (0, shift):
            buf = torch.zeros(rows * (heads * hd + pad) + pad, dtype=t, device="cuda")
            v = buf[pad:].view(rows, heads * hd + pad)[:, :heads * hd]
            v.copy_(x)
            device.qk_norm_rope(nebw.Heads.of(v, heads, gamma=gamma), None, rows, hd, rope=h,
                                pos=pos)
            device.sync()
            outs.append(v.clone())
        # the two sum a head's squares in different orders
        a, b = outs[0].double(), outs[1].double()
        assert ((a - b).abs() <= 2 * half_step(t) * a.abs() + (hd + 8) * U * 8).all()
    finally:
        device.release_weight(h)


def test_head_norm_without_rotation_and_one_side(device):
    import nebw
    rows, heads, hd = 50, 4, 64
    g = gen(5)
    x = torch.randn(rows, heads * hd, generator=g, device="cuda").to(torch.bfloat16)
    gamma = torch.randn(hd, generator=g, device="cuda")
    out = torch.empty_like(x)
    for q, k in ((1, 0), (0, 1)):
        out.zero_()
        side = nebw.Heads.of(x, heads, out=out, gamma=gamma)
        device.qk_norm_rope(side if q else None, side if k else None, rows, hd, eps=1e-6)
        device.sync()
        assert_close(out, *heads_reference(x, heads, hd, [], 1.0, None, False, 1, gamma, None,
                                           1e-6))


def test_head_rows_of_zeros_and_infinities(device):
    """A head of zeros stays finite under eps; a NaN or infinity stays in its head."""
    import nebw
    rows, heads, hd = 6, 3, 64
    g = gen(6)
    x = torch.randn(rows, heads * hd, generator=g, device="cuda").to(torch.bfloat16)
    x[0] = 0
    x[2, hd + 3] = float("inf")
    x[4, 2 * hd + 9] = float("nan")
    gamma = torch.ones(hd, device="cuda")
    out = torch.empty_like(x)
    inv, scale = nebw.rope_freqs(10000.0, hd)
    h = device.stage_rope(inv, 16, scale)
    try:
        pos = torch.arange(rows, device="cuda").int()
        device.qk_norm_rope(nebw.Heads.of(x, heads, out=out, gamma=gamma), None, rows, hd, rope=h,
                            pos=pos)
        device.sync()
        assert (out[0] == 0).all()
        fine = torch.isfinite(out.view(rows, heads, hd)).all(-1)
        want = torch.ones(rows, heads, dtype=torch.bool, device="cuda")
        want[2, 1] = want[4, 2] = False
        assert torch.equal(fine, want)
    finally:
        device.release_weight(h)


@pytest.mark.parametrize("heads", [2, 16])  # several rows a warp, and one
def test_heads_live_rows_and_bad_positions(device, heads):
    """Rows behind the live count stay; a position outside the table is
    reported and the nearest entry used."""
    import nebw
    rows, hd = 40, 64
    g = gen(7)
    x = torch.randn(rows, heads * hd, generator=g, device="cuda").to(torch.bfloat16)
    inv, scale = nebw.rope_freqs(10000.0, hd)
    h = device.stage_rope(inv, 100, scale)
    try:
        for live in (0, 1, 17, 40, 99, -3):
            out = torch.full_like(x, 7.0)
            n = torch.tensor([live], dtype=torch.int32, device="cuda")
            pos = torch.arange(rows, device="cuda").int()
            live = max(0, min(live, rows))
            pos[live:] = 1 << 30  # positions of rows that are not there are not looked at
            device.rope(nebw.Heads.of(x, heads, out=out), None, rows, hd, h, pos, rows_dev=n)
            device.sync()
            assert (out[live:] == 7.0).all()
            assert_close(out[:live], *heads_reference(x[:live], heads, hd, inv, scale, pos[:live],
                                                      False))
        for bad, used in ((-1, 0), (100, 99), (2 ** 31 - 1, 99), (-2 ** 31, 0)):
            out = torch.empty_like(x)
            pos = torch.arange(rows, device="cuda").int()
            pos[11] = bad
            device.rope(nebw.Heads.of(x, heads, out=out), None, rows, hd, h, pos)
            with pytest.raises(nebw.NebwError, match="position"):
                device.sync()
            pos[11] = used
            assert_close(out, *heads_reference(x, heads, hd, inv, scale, pos, False))
    finally:
        device.release_weight(h)


def test_heads_past_32_bits(device):
    """Rows whose element offsets need more than 32 bits."""
    import nebw
    rows, stride, hd = 36000, 1 << 17, 64
    buf = torch.empty(rows, stride, dtype=torch.bfloat16, device="cuda")  # 9.4 GB
    x = buf[:, 5 * hd:6 * hd]
    x.copy_(torch.randn(rows, hd, generator=gen(14), device="cuda"))
    before = x.clone()
    inv, scale = nebw.rope_freqs(10000.0, hd)
    h = device.stage_rope(inv, rows)
    pos = torch.arange(rows, device="cuda").int()
    device.rope(nebw.Heads.of(x, 1), None, rows, hd, h, pos)
    device.sync()
    assert_close(x, *heads_reference(before, 1, hd, inv, scale, pos, False))
    device.release_weight(h)


def test_rope_table_far_positions(device):
    """Angles of far positions keep their fraction: 2^20 positions against 64 bits."""
    import nebw
    max_pos, hd = 1 << 20, 64
    inv, scale = nebw.rope_freqs(500000.0, hd, "bands", factor=8.0, orig_len=8192)
    h = device.stage_rope(inv, max_pos, scale)
    try:
        pos = torch.tensor([0, 1, 8191, 65537, max_pos - 2, max_pos - 1], device="cuda").int()
        x = torch.randn(len(pos), hd, generator=gen(8), device="cuda")
        out = torch.empty_like(x)
        device.rope(nebw.Heads.of(x, 1, out=out), None, len(pos), hd, h, pos)
        device.sync()
        assert_close(out, *heads_reference(x, 1, hd, inv, scale, pos, False))
    finally:
        device.release_weight(h)


def test_rope_equals_the_models_own_rotation(device):
    """The half layout over the whole head is what the rotary models apply: the
    frequency set of nebw_rope_freqs given to a model encodes as its theta does."""
    import ctypes as C

    import nebw
    from nebw import synth
    w = synth.config_weights(synth.CONFIGS["nomic-base"], layers=1)
    lens = np.array([40, 3, 64], np.int32)
    ids, _mask = synth.make_tokens(3, 64, lens, seed=9)
    model = nebw.Model.from_weights(device, w, max_seq_len=64)
    try:
        want = model.encode(ids, lens)
        inv, scale = nebw.rope_freqs(w.rope_theta, w.head_dim)
        assert scale == 1.0
        assert nebw.lib().nebw_model_set_rope_freq(
            model.h, inv.ctypes.data_as(C.POINTER(C.c_double)), len(inv)) == 0
        # the two pow forms differ by an ulp of double: the fp32 tables may
        # differ by one rounding in rare entries
        assert np.abs(model.encode(ids, lens) - want).max() <= 1e-5
    finally:
        model.close()


def test_row_positions(device):
    lens = torch.tensor([5, 1, 300, 64], dtype=torch.int32, device="cuda")
    n, off = torch.empty_like(lens), torch.empty(5, dtype=torch.int32, device="cuda")
    device.pack_offsets(lens, 4, 300, n, off)
    pos = torch.full((400,), -7, dtype=torch.int32, device="cuda")
    device.row_positions(off, n, 4, 300, pos)
    device.sync()
    want = torch.cat([torch.arange(int(v)) for v in lens.cpu()] + [torch.full((30,), -7)])
    assert torch.equal(pos.cpu(), want.int())


def test_row_positions_stop_at_the_bound(device):
    """Lengths past max_len are cut there, and an empty batch has no addresses."""
    off = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    n = torch.tensor([290, 7], dtype=torch.int32, device="cuda")
    pos = torch.full((400,), -7, dtype=torch.int32, device="cuda")
    device.row_positions(off, n, 2, 258, pos)
    empty = off[:0].clone()
    device.row_positions(empty, empty, 0, 258, empty)
    device.sync()
    want = torch.full((400,), -7)
    want[:258], want[300:307] = torch.arange(258), torch.arange(7)
    assert torch.equal(pos.cpu(), want.int())


@pytest.mark.parametrize("heads,hd", [(4, 64), (8, 32)])
@pytest.mark.parametrize("norm", [1, 2])
def test_normed_heads_ahead_of_attention(device, heads, hd, norm):
    """The documented way: the softmax's 1/sqrt(head_dim) in the query norm's
    weight and bias, the Q|K|V rows in place, then the framework's attention."""
    import nebw
    lens = [70, 1, 128, 33]
    T, H, g = sum(lens), heads * hd, gen(60 + hd + norm)
    qkv = torch.randn(T, 3 * H, generator=g, device="cuda").bfloat16()
    gam = [1 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)]
    bet = [0.3 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)]
    by = 1.0 / math.sqrt(hd)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    off, pos = torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty_like(qkv[:, 0]).int()
    device.pack_offsets(n, 4, 128, n, off)
    device.row_positions(off, n, 4, 128, pos)
    inv, _ = nebw.rope_freqs(10000.0, hd)
    table = device.stage_rope(inv, 128)
    side = [heads_reference(qkv[:, i * H:(i + 1) * H], heads, hd, inv, 1.0, pos, False, norm,
                            gam[i], bet[i], 1e-6)[0].view(T, heads, hd) for i in range(2)]
    v = qkv[:, 2 * H:].double().view(T, heads, hd)

    def attention(scale):
        """ctx in 64 bits, the sum of p |v|, and the most a logit is off."""
        out, size, most, at = [], [], [], 0
        for m in lens:
            s = slice(at, at + m)
            p = torch.softmax(scale * torch.einsum("qhd,khd->hqk", side[0][s], side[1][s]), -1)
            terms = scale * torch.einsum("qhd,khd->hqk", side[0][s].abs(), side[1][s].abs())
            out.append(torch.einsum("hqk,khd->qhd", p, v[s]))
            size.append(torch.einsum("hqk,khd->qhd", p, v[s].abs()))
            most.append(terms.amax(-1).t()[:, :, None].expand(m, heads, hd))
            at += m
        return [torch.cat(t).reshape(T, H) for t in (out, size, most)]

    q = nebw.Heads.of(qkv[:, :H], heads, gamma=gam[0] * by, beta=bet[0] * by)
    k = nebw.Heads.of(qkv[:, H:2 * H], heads, gamma=gam[1], beta=bet[1])
    device.qk_norm_rope(q, k, T, hd, norm=norm, eps=1e-6, rope=table, pos=pos)
    ctx = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    device.attention(qkv, T, off, n, 4, 128, heads, hd, ctx)
    device.sync()
    want, size, most = attention(by)
    # q and k are rounded to bf16 (2^-8 each of every term of a logit), which moves
    # a probability and its sum by that exponent each; p is rounded to bf16
    # (2^-8), the fp32 steps are below a tenth of it, and ctx is rounded
    tol = (torch.expm1(2 * 2.0 ** -7 * most) + 1.2 * 2.0 ** -8) * size + 2.0 ** -8 * want.abs()
    assert ((ctx.double() - want).abs() <= tol).all()
    # without the scale the result would be another one
    far = (attention(1.0)[0] - want).abs()
    assert (far > 2 * tol).float().mean() > 0.2
    device.release_weight(table)


@pytest.mark.parametrize("off,lens", [
    ([0, 90], [5, 20]),          # past the end
    ([-3, 40], [5, 20]),         # before the start
    ([2 ** 31 - 1, 40], [5, 20]), ([-2 ** 31, 40], [5, 20]),
    ([0, 100], [5, 1]),
])
def test_row_positions_outside_the_rows(device, off, lens):
    """Offsets that leave pos are reported; what lies in it is written, what lies
    around it (with room on both sides) stays."""
    import nebw
    buf = torch.full((300,), -7, dtype=torch.int32, device="cuda")
    pos = buf[100:200]
    o, n = (torch.tensor(v, device="cuda").int() for v in (off, lens))
    device.row_positions(o, n, 2, 64, pos)
    with pytest.raises(nebw.NebwError, match="packed row") as e:
        device.sync()
    assert e.value.code == 5
    want = torch.full((300,), -7)
    for a, m in zip(off, lens):
        for s in range(m):
            if 0 <= a + s < 100:
                want[100 + a + s] = s
    assert torch.equal(buf.cpu(), want.int())
    device.sync()  # reported once
    with pytest.raises(ValueError):  # fewer entries than said
        device.row_positions(o, n, 2, 64, pos, rows=101)
    with pytest.raises(nebw.NebwError, match="rows"):
        device.row_positions(o, n, 2, 64, pos, rows=-1)


def test_row_positions_by_address_and_of_whole_sequences(device):
    """The entry point without a row count writes as many as the sequences can
    have; an address comes with its number."""
    import nebw
    off, n = (torch.tensor(v, device="cuda").int() for v in ([0, 5], [5, 8]))
    pos = torch.full((20,), -7, dtype=torch.int32, device="cuda")
    want = torch.cat([torch.arange(5), torch.arange(8), torch.full((7,), -7)]).int()
    rc = nebw.lib().nebw_row_positions(device.h, off.data_ptr(), n.data_ptr(), 2, 8,
                                       pos.data_ptr(), nebw.CUDA_STREAM_LEGACY)
    device.sync()
    assert rc == 0 and torch.equal(pos.cpu(), want)
    pos.fill_(-7)
    device.row_positions(off, n, 2, 8, pos.data_ptr(), rows=13)
    device.sync()
    assert torch.equal(pos.cpu(), want)


def test_heads_refusals(device):
    import nebw
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    gamma = torch.ones(64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    inv, _ = nebw.rope_freqs(10000.0, 64)
    h = device.stage_rope(inv, 16)
    hd = nebw.Heads.of(x, 2, gamma=gamma)

    def refused(word, fn, *a, **k):
        with pytest.raises(nebw.NebwError, match=word) as e:
            fn(*a, **k)
        assert e.value.code == 1

    try:
        refused("unknown rotary", device.rope, hd, None, 4, 64, h + 1000, pos)
        refused("without a rotary", device.rope, hd, None, 4, 64, 0, pos)
        refused("without positions", device.rope, hd, None, 4, 64, h, None)
        refused("more than head_dim", device.rope, hd, None, 4, 32, h, pos)
        p = x.data_ptr()
        raw = nebw.Heads(p, p, 128, 128, 2)
        refused("head_dim 258", device.rope, raw, None, 4, 258, h, pos)
        refused("head_dim 63", device.rope, hd, None, 4, 63, h, pos)
        refused("layout", device.rope, hd, None, 4, 64, h, pos, layout=2)
        refused("no heads", device.rope, None, None, 4, 64, h, pos)
        refused("rows", device.rope, hd, None, -1, 64, h, pos)
        refused("rows", device.rope, raw, None, 1 << 31, 64, h, pos.data_ptr())
        refused("head norm", device.qk_norm_rope, hd, None, 4, 64, norm=0)
        refused("head norm", device.qk_norm_rope, hd, None, 4, 64, norm=3)
        refused("eps", device.qk_norm_rope, hd, None, 4, 64, eps=float("nan"))
        refused("without its bias", device.qk_norm_rope, hd, None, 4, 64, norm=2)
        refused("without its weight", device.qk_norm_rope, nebw.Heads.of(x, 2), None, 4, 64)
        refused("stride", device.rope, raw, None, 4, 128, h, pos)
        refused("one row stride", device.rope, nebw.Heads(p, p, 128, 192, 2), None, 4, 64, h, pos)
        refused("aligned", device.rope, nebw.Heads(p + 1, p, 128, 128, 2), None, 4, 64, h, pos)
        refused("null query", device.rope, nebw.Heads(None, p, 128, 128, 2), None, 4, 64, h, pos)
        refused("null key", device.rope, hd, nebw.Heads(p, None, 128, 128, 2), 4, 64, h, pos)
        refused("dtype", device.rope, nebw.Heads(p, p, 128, 128, 2), None, 4, 64, h, pos, dtype=2)
        refused("frequencies", device.stage_rope, np.ones(129), 16)
        refused("positions", device.stage_rope, inv, 0)
        refused("positions", device.stage_rope, inv, 1 << 40)
        refused("scale", device.stage_rope, inv, 16, float("nan"))
        refused("not finite", device.stage_rope, np.array([1.0, np.inf]), 16)
        assert torch.equal(x, torch.zeros_like(x))
        for few in ((5, 64, h, pos), (4, 66, h, pos), (4, 64, h, pos[:3])):  # what is not there
            with pytest.raises(ValueError):
                device.rope(hd, None, *few)
        device.rope(hd, None, 0, 64, h, None)  # no rows: nothing to do
        device.rope(nebw.Heads.of(x[:0].clone(), 2), None, 0, 64, h, pos[:0].clone())
        device.sync()
    finally:
        device.release_weight(h)
    refused("unknown rotary", device.rope, hd, None, 4, 64, h, pos)


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------

def route_reference(logits, k, sigmoid=False, renorm=False, scale=1.0):
    """ids, weights (64 bits), group_off, row_src, row_dst by the definition."""
    x = logits.double().cpu().numpy()
    rows, experts = x.shape
    ids = np.full((rows, k), -1, np.int32)
    w = np.zeros((rows, k))
    for t in range(rows):
        able = [e for e in range(experts) if x[t, e] > -np.inf]
        best = sorted(able, key=lambda e: (-x[t, e], e))[:k]
        if not best:
            continue
        top = x[t, best[0]]
        with np.errstate(over="ignore", invalid="ignore"):
            p = {e: 1 / (1 + np.exp(-x[t, e])) if sigmoid else
                 1.0 if x[t, e] == top else np.exp(x[t, e] - top) for e in able}
        total = sum(p[e] for e in best) if renorm else 1.0 if sigmoid else sum(p.values())
        for j, e in enumerate(best):
            ids[t, j], w[t, j] = e, scale * p[e] / total if total else 0.0
    flat = ids.reshape(-1)
    order = [i for e in range(experts) for i in np.flatnonzero(flat == e)]
    dst = np.full(rows * k, -1, np.int32)
    dst[order] = np.arange(len(order))
    off = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(experts)])])
    return ids, w, off.astype(np.int32), np.array(order, np.int64) // k, dst.reshape(rows, k)


class Routing:
    """The outputs of one call, filled with what must stay where nothing is written."""

    def __init__(self, rows, experts, k):
        import nebw
        self.shape = rows, experts, k
        self.ids = torch.full((rows, k), -77, dtype=torch.int32, device="cuda")
        self.weights = torch.full((rows, k), -77.0, device="cuda")
        self.off = torch.full((experts + 1,), -77, dtype=torch.int32, device="cuda")
        self.src = torch.full((rows * k,), -77, dtype=torch.int32, device="cuda")
        self.dst = torch.full((rows, k), -77, dtype=torch.int32, device="cuda")
        self.ws = torch.full((nebw.moe_route_workspace(rows, experts, k) // 4,), -77,
                             dtype=torch.int32, device="cuda")

    def run(self, device, logits, **kw):
        rows, experts, k = self.shape
        device.moe_route(logits, rows, experts, k, self.ids, self.weights, self.off, self.src,
                         self.dst, self.ws, **kw)
        return self

    def check(self, want, live=None):
        ids, w, off, src, dst = want
        rows = self.shape[0] if live is None else live
        np.testing.assert_array_equal(self.ids.cpu().numpy()[:rows], ids)
        np.testing.assert_array_equal(self.off.cpu().numpy(), off)
        np.testing.assert_array_equal(self.src.cpu().numpy()[:len(src)], src)
        np.testing.assert_array_equal(self.dst.cpu().numpy()[:rows], dst)
        got = self.weights.double().cpu().numpy()[:rows]
        # exp to 2 ulp at an argument rounded to 2^-24 of up to ~100, a sum
        # of up to 512 terms, a divide, a product
        np.testing.assert_allclose(got, w, rtol=700 * U, atol=1e-37)
        assert (self.ids.cpu().numpy()[rows:] == -77).all()
        assert (self.weights.cpu().numpy()[rows:] == -77).all()
        assert (self.dst.cpu().numpy()[rows:] == -77).all()
        assert (self.src.cpu().numpy()[len(src):] == -77).all()


ROUTE_CASES = [
    # rows, experts, top_k
    (1, 1, 1), (1, 8, 2), (5, 4, 4), (31, 6, 2), (100, 8, 2), (300, 16, 16), (64, 64, 8),
    (33, 60, 6), (129, 128, 4), (200, 200, 8), (70, 256, 8), (40, 512, 16), (513, 8, 2),
    (1500, 64, 8), (2049, 33, 1),
    # around where one block hands over to two kernels, and one block with
    # more rows than it places at once
    (190, 64, 8), (220, 64, 8), (1000, 8, 2), (1001, 8, 2), (1990, 4, 1),
]


@pytest.mark.parametrize("rows,experts,k", [(170001, 4, 1), (131071, 64, 8), (400003, 8, 2)])
def test_route_many_rows(device, rows, experts, k):
    """Many rows (also more than a block places at once) against the stable sort."""
    x = torch.randn(rows, experts, generator=gen(rows), device="cuda").bfloat16()
    r = Routing(rows, experts, k).run(device, x, renorm=True)
    device.sync()
    ids = x.float().sort(dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.ids.long(), ids)
    order = ids.reshape(-1).sort(stable=True)
    edges = torch.arange(experts + 1, device="cuda")
    assert torch.equal(r.off.long(), torch.searchsorted(order.values, edges))
    assert torch.equal(r.src.long(), order.indices // k)
    place = torch.empty_like(order.indices)
    place[order.indices] = torch.arange(rows * k, device="cuda")
    assert torch.equal(r.dst.long().reshape(-1), place)
    want = torch.softmax(x.double().gather(1, ids), 1)
    assert ((r.weights.double() - want).abs() <= 100 * U * want).all()


@pytest.mark.parametrize("score,renorm", [(0, False), (0, True), (1, False), (1, True)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,experts,k", ROUTE_CASES)
def test_route_matches_definition(device, rows, experts, k, dtype, score, renorm):
    x = (2 * torch.randn(rows, experts, generator=gen(rows + experts + k), device="cuda")).to(
        TYPES[dtype])  # bf16: many ties
    r = Routing(rows, experts, k).run(device, x, score=score, renorm=renorm, scale=2.5)
    device.sync()
    r.check(route_reference(x, k, score == 1, renorm, 2.5))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_route_ties_masks_and_odd_values(device, dtype):
    """Equal logits go to the lower expert (-0 and +0 are equal); -inf and NaN
    are never chosen; a row without any expert has no place; +inf wins."""
    inf, nan, low = math.inf, math.nan, torch.finfo(TYPES[dtype]).min
    x = torch.tensor([
        [0.0, -0.0, 0.0, -0.0, 0.0, 0.0],
        [-0.0, 0.0, -0.0, 0.0, -1.0, -1.0],
        [-inf, -inf, 2.0, -inf, -inf, 2.0],
        [-inf, 1.0, -inf, -inf, -inf, -inf],
        [-inf] * 6,
        [nan] * 6,
        [nan, 1.0, nan, 3.0, nan, 2.0],
        [low, low, -inf, low, 0.0, low],
        [low] * 6,
        [inf, 1.0, inf, 2.0, -inf, 0.0],
        [inf] * 6,
        [-200.0, -150.0, -300.0, -250.0, -400.0, -120.0],
        [200.0, 150.0, 300.0, 250.0, 400.0, 120.0],
        [1.0, 2.0, 3.0, 3.0, 2.0, 1.0],
    ], device="cuda").to(TYPES[dtype])
    for score in (0, 1):
        for renorm in (False, True):
            r = Routing(len(x), 6, 3).run(device, x, score=score, renorm=renorm)
            device.sync()
            w = r.weights
            assert torch.isfinite(w).all()
            ids, want, off, src, dst = route_reference(x, 3, score == 1, renorm)
            big = torch.isinf(x).logical_and(x > 0).any(1).cpu().numpy()
            if score == 0:  # with an infinite logit: shared among the infinite ones
                assert w[9].tolist() == pytest.approx([0.5, 0.5, 0.0])
                share = 1 / 3 if renorm else 1 / 6
                assert w[10].tolist() == pytest.approx([share] * 3)
                want[big] = w.double().cpu().numpy()[big]
            # sigmoid of -120 and below: fp32 knows no smaller sum
            tiny = score == 1 and renorm
            if tiny:
                want[11] = w.double().cpu().numpy()[11]
                assert (w[11] >= 0).all() and float(w[11].sum()) <= 1.0 + 4 * U
            r.check((ids, np.where(np.abs(want) < 2e-38, 0, want) if score else want, off, src,
                     dst))


@pytest.mark.parametrize("scale", [1.0, 2.5])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_route_sigmoid_shares_of_very_low_logits(device, dtype, scale):
    """Divided by the sum of the chosen, sigmoids that fp32 cannot hold are
    still shares of one; a row of lowest values has no share to give."""
    low = torch.finfo(TYPES[dtype]).min
    x = torch.cat([
        torch.tensor([[-200.0, -150.0, -300.0, -250.0, -400.0, -120.0],
                      [-700.0, low, -708.0, low, -900.0, low], [low] * 6,
                      [-712.0, -712.0, -3e4, low, low, low], [low, -1.0, low, low, low, 3.0], [-math.inf, -90.0, -math.inf, -91.0, -92.0, 0.0],
                      [-math.inf, -90.0, -math.inf, -90.5, -92.0, -math.inf]], device="cuda"),
        # around where exp(-x) leaves fp32, and its reciprocal the normal range
        -torch.arange(80.0, 110.0, 0.125, device="cuda").reshape(-1, 6)]).to(TYPES[dtype])
    for k in (1, 2, 3):
        r = Routing(len(x), 6, k).run(device, x, score=1, renorm=True, scale=scale)
        device.sync()
        v = x.double()
        best = v.sort(dim=1, descending=True, stable=True)
        top, ids = best.values[:, :k], best.indices[:, :k]
        there = top > -math.inf
        # sigmoid(v) / sum = exp(v - log(1 + e^v)) / sum, from the logarithms
        want = scale * torch.softmax(torch.nn.functional.logsigmoid(top), 1) * there
        want = torch.where(top[:, :1] > -709.78, want, 0.0)
        assert torch.equal(r.ids, torch.where(there, ids, -1).int())
        # as Routing.check: two exp of arguments to ~100, sums, quotients, a product
        got = r.weights.double()
        assert ((got - want).abs() <= 700 * U * want + 1e-37).all(), (got, want)


@pytest.mark.parametrize("rows", [1200, 700])  # two kernels, and one block
def test_route_live_rows(device, rows):
    experts, k = 16, 2
    x = torch.randn(rows, experts, generator=gen(3), device="cuda")
    for live in (0, 1, 31, 32, 511, 513, rows - 1, rows, 5000, -1):
        n = torch.tensor([live], dtype=torch.int32, device="cuda")
        r = Routing(rows, experts, k).run(device, x, rows_dev=n)
        device.sync()
        live = max(0, min(live, rows))
        r.check(route_reference(x[:live], k), live)


def test_route_strided_logits_and_repeat(device):
    """A padded product's rows; the same call twice gives the same bits, also
    with another call's leavings in the workspace."""
    rows, experts, k = 900, 6, 2
    wide = torch.randn(rows, 8, generator=gen(4), device="cuda")
    wide[:, 6:] = 100.0  # padding columns are not looked at
    r = Routing(rows, experts, k)
    r.run(device, wide[:, :6])
    device.sync()
    r.check(route_reference(wide[:, :6].contiguous(), k))
    first = [t.clone() for t in (r.ids, r.weights, r.off, r.src, r.dst)]
    r.run(device, -wide[:, :6])
    r.run(device, wide[:, :6])
    device.sync()
    assert all(torch.equal(a, b) for a, b in zip(first, (r.ids, r.weights, r.off, r.src, r.dst)))


def test_route_empty_and_refusals(device):
    import nebw
    r = Routing(40, 8, 2)  # room for what the calls below ask for
    x = torch.zeros(4, 8, device="cuda")
    device.moe_route(x[:0], 0, 8, 2, r.ids, r.weights, r.off, r.src, r.dst, r.ws)
    device.sync()
    assert (r.off == 0).all() and (r.ids == -77).all()

    def refused(word, logits=x, rows=4, experts=8, k=2, ids=r.ids, ws=r.ws, **kw):
        with pytest.raises(nebw.NebwError, match=word) as e:
            device.moe_route(logits, rows, experts, k, ids, r.weights, r.off, r.src, r.dst, ws,
                             **kw)
        assert e.value.code == 1

    refused("top_k", k=0)
    refused("top_k", k=9)
    refused("rows", rows=-1)
    refused("score", score=2)
    refused("scale", scale=float("inf"))
    refused("null routing", ids=None)
    few = r
    r = Routing(1 << 20, 8, 2)
    refused("workspace", logits=torch.zeros(1 << 20, 8, device="cuda"), ids=r.ids, ws=x,
            rows=1 << 20)
    with pytest.raises(ValueError):  # fewer values than the call writes
        device.moe_route(torch.zeros(99, 8, device="cuda"), 99, 8, 2, few.ids, r.weights, r.off,
                         r.src, r.dst, r.ws)
    with pytest.raises(ValueError):
        device.moe_route(x, 5, 8, 2, r.ids, r.weights, r.off, r.src, r.dst, r.ws)
    wide = torch.zeros(1, 600, device="cuda")
    r.off = torch.zeros(514, dtype=torch.int32, device="cuda")
    refused("experts", logits=wide, rows=1, experts=513)
    with pytest.raises(ValueError):
        device.moe_route(x.t(), 8, 4, 2, r.ids, r.weights, r.off, r.src, r.dst, r.ws)
    with pytest.raises(TypeError):
        device.moe_route(x.half(), 4, 8, 2, r.ids, r.weights, r.off, r.src, r.dst, r.ws)


# ---------------------------------------------------------------------------
# grouped products
# ---------------------------------------------------------------------------

def gelu8_64(v):
    """The reference's degree-8 polynomial, in 64 bits."""
    u = v.abs().clamp(max=4.0)
    p = torch.full_like(u, -7.2340282171e-05)
    for c in (1.8179518005e-03, -1.7707383379e-02, 8.4577147641e-02, -1.9228671834e-01,
              9.8431124458e-02, 3.6137852062e-01, -4.9454128936e-01, -1.3007010117e-04):
        p = p * u + c
    return v.clamp(min=0) + p


def grouped_reference(a, w, off, src, bias, gated, act):
    """(value, bound of the fp32 error) of the grouped product, in 64 bits."""
    a = a.double()
    if src is not None:
        a = a[src.long()]
    K = a.shape[1]
    vals, errs = [], []
    for e in range(w.shape[0]):
        x = a[off[e]:off[e + 1]]
        we = w[e].double()
        v, size = x @ we, x.abs() @ we.abs()
        if bias is not None:
            v, size = v + bias[e].double(), size + bias[e].double().abs()
        vals.append(v)
        # K products and adds, each off by at most two units of the running sum
        errs.append((K + 2) * 2 * U * size)
    v, err = torch.cat(vals), torch.cat(errs)
    if gated:
        f = v.shape[1] // 2
        u, g, eu, eg = v[:, :f], v[:, f:], err[:, :f], err[:, f:]
        s = g * torch.sigmoid(g) if act == 0 else g * torch.special.ndtr(g)
        # |act'| <= 1.13; erf gelu is off by 7e-7, silu by 2^-19 of itself
        es = 1.13 * eg + (s.abs() * 2.0 ** -19 if act == 0 else 7e-7 + 4 * U * g.abs())
        return u * s, s.abs() * eu + (u.abs() + eu) * es + U * (u * s).abs()
    if act == 1:
        return gelu8_64(v), 1.13 * err + 16 * U * (1 + v.abs())
    if act == 2:
        return v * torch.special.ndtr(v), 1.13 * err + 7e-7 + 4 * U * v.abs()
    return v, err


def groups(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


GROUP_CASES = [
    # sizes of the groups, K, N
    ([1], 64, 8),
    ([1, 0, 0, 2], 64, 64),
    ([0, 0, 3], 72, 24),
    ([5, 5, 5, 5, 5, 5, 5, 5], 200, 128),
    ([127, 128, 129, 1], 128, 256),
    ([0, 300, 0, 41], 384, 520),
    ([255, 256, 257], 256, 512),
    ([700], 1000, 256),
    ([1] * 40 + [0] * 20 + [33], 128, 128),
    ([64, 17, 1, 0, 290, 3], 512, 1536),
    ([20, 31, 32, 33, 63, 64, 65, 96], 768, 768),
    ([3000, 1, 0, 1200], 256, 1024),
    # several tiles a block, with part tiles among them: one CTA, and a pair
    ([130, 3, 257, 1, 90, 128, 0, 200] * 10, 192, 1024),
    ([2100, 1, 900, 513, 40, 2500] * 2, 192, 1536),
    # small groups but for one, which the smaller tiles cut in three
    ([300, 1, 2, 0, 5, 3, 1, 0, 2, 6], 128, 520),
]
EPILOGUES = [  # gated, act, output
    (False, 0, "bf16"), (False, 0, "f32"), (False, 1, "bf16"), (False, 2, "bf16"),
    (True, 0, "bf16"), (True, 1, "bf16"),
]


@pytest.mark.parametrize("gated,act,out", EPILOGUES)
@pytest.mark.parametrize("gather,bias", [(False, False), (True, True)])
@pytest.mark.parametrize("sizes,K,N", GROUP_CASES)
def test_grouped_product_matches_64_bits(device, sizes, K, N, gather, bias, gated, act, out):
    import nebw
    if gated and N % 64:
        N = (N + 63) // 64 * 64
    E, M = len(sizes), sum(sizes)
    g = gen(M + K + N)
    off = groups(sizes)
    w = (torch.randn(E, K, N, generator=g, device="cuda") * 1.5 / math.sqrt(K)).bfloat16()
    a_rows = max(1, M // 2) if gather else M
    a = torch.randn(a_rows, K, generator=g, device="cuda").bfloat16()
    src = torch.randint(0, a_rows, (M,), generator=g, device="cuda").int() if gather else None
    b = 0.3 * torch.randn(E, N, generator=g, device="cuda") if bias else None
    n_out = N // 2 if gated else N
    rows = M + 3  # the bound may be more than the groups hold
    c = torch.full((rows, n_out), 7.0, dtype=TYPES[out], device="cuda")
    if gather:
        src_in = torch.cat([src, src.new_full((3,), 1 << 30)])
        a_in = a
    else:
        src_in = None
        a_in = torch.cat([a, a.new_full((3, K), math.nan)])
    h = device.stage_experts(w, gated=gated)
    try:
        device.gemm_grouped(h, a_in, a_in.shape[0], torch.from_numpy(off).cuda(), rows, K, N, c,
                            row_src=src_in, bias=b, act=act,
                            c_dtype=nebw.BF16 if out == "bf16" else nebw.F32)
        device.sync()
        assert (c[M:] == 7.0).all()
        assert_close(c[:M], *grouped_reference(a, w, off, src, b, gated, act))
    finally:
        device.release_weight(h)


@pytest.mark.parametrize("K", [128, 136, 320, 1024, 1536, 1544, 2048, 4000])
def test_grouped_fp32_output_over_long_products(device, K):
    """fp32 output keeps K in parts: up to four of half tiles, two of whole ones.

    The tensor core cuts its sum once a step of 16, by half a unit (2^-24 of
    the running sum) on average.  The running sum of independent products grows
    as the root of the steps, so S steps of a part lose S * 2^-24 * 2 / 3 of
    the part, and parts of random sign lose the same of their sum.  At 2048
    that is 1.3e-6; one part of K would lose four times as much."""
    import nebw
    sizes, N = [300, 0, 129, 1, 700, 128, 64], 520
    off, E, M = groups(sizes), 7, sum(sizes)
    g = gen(K)
    w = (torch.randn(E, K, N, generator=g, device="cuda") / math.sqrt(K)).bfloat16()
    a = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    c = torch.full((M, N), 7.0, device="cuda")
    h = device.stage_experts(w)
    try:
        device.gemm_grouped(h, a, M, torch.from_numpy(off).cuda(), M, K, N, c, c_dtype=nebw.F32)
        device.sync()
        want, err = grouped_reference(a, w, off, None, None, False, 0)
        assert_close(c, want, err)
        parts = 4 if K > 1536 else 2
        steps = -(-K // (64 * parts)) * 4
        lost = ((c.double() - want).norm() / want.norm()).item()
        assert lost < steps * 2.0 ** -24 * 2 / 3 + 4 * U
    finally:
        device.release_weight(h)


@pytest.mark.parametrize("signed", [False, True])
@pytest.mark.parametrize("K,rows,parts", [
    (1024, 700, 2), (1536, 700, 2), (1544, 700, 4), (2048, 700, 4), (4000, 700, 4),
    (1024, 60, 4), (2048, 60, 4), (16384, 300, 4)])
def test_grouped_fp32_output_loses_its_part_of_one_sum(device, K, rows, parts, signed):
    """P parts of K lose about 1/P of what one accumulator over all of K loses:
    each step of 16 cuts by a share of the running sum, which in a part is as
    long on average as its share of the steps, and the adding of P parts is exact
    next to that.  nebw_gemm keeps one accumulator.  Half the parts would lose
    twice as much: the bound lies between, at sqrt(2) / P.  Products of one sign,
    whose cuts all go one way, show it as well."""
    import nebw
    N, g = 264, gen(K + rows)
    a = torch.randn(rows, K, generator=g, device="cuda")
    w = torch.randn(1, K, N, generator=g, device="cuda") / math.sqrt(K)
    if signed:
        a, w = a.abs(), w.abs()
    a, w = a.bfloat16(), w.bfloat16()
    want = a.double() @ w[0].double()
    one = device.stage_weight(w[0].view(torch.int16).cpu().numpy().view(np.uint16))
    many = device.stage_experts(w)
    lost = []
    for grouped in (False, True):
        c = torch.empty(rows, N, device="cuda")
        if grouped:
            device.gemm_grouped(many, a, rows, torch.tensor([0, rows], device="cuda").int(), rows, K,
                                N, c, c_dtype=nebw.F32)
        else:
            device.gemm(one, a, rows, K, N, c, c_dtype=nebw.F32)
        device.sync()
        lost.append(((c.double() - want).norm() / want.norm()).item())
    assert lost[1] < math.sqrt(2) / parts * lost[0], lost
    # and one unit of the running sum a step at most
    assert lost[1] < K / (16 * parts) * 2.0 ** -23, lost
    device.release_weight(one)
    device.release_weight(many)


def test_grouped_product_of_more_tiles_than_are_looked_up(device):
    """512 experts of a row each, 19 column tiles: over 128 tiles a block."""
    E, K, N = 512, 64, 4864
    w = torch.randn(E, K, N, generator=gen(9), device="cuda").bfloat16()
    a = torch.randn(E, K, generator=gen(10), device="cuda").bfloat16()
    h = device.stage_experts(w)
    c = torch.empty(E, N, dtype=torch.bfloat16, device="cuda")
    off = torch.arange(E + 1, device="cuda").int()
    device.gemm_grouped(h, a, E, off, E, K, N, c)
    device.sync()
    want = torch.einsum("ek,ekn->en", a.double(), w.double())
    size = torch.einsum("ek,ekn->en", a.double().abs(), w.double().abs())
    assert_close(c, want, (K + 2) * 2 * U * size)
    device.release_weight(h)


def test_grouped_product_does_not_mix_groups(device):
    """A NaN row stays in its own row of C, and an expert's NaN weights in its
    group, also inside a tile that reaches into the next group."""
    sizes, K, N = [10, 20, 30], 128, 256
    off, M = groups(sizes), 60
    g = gen(1)
    w = torch.randn(3, K, N, generator=g, device="cuda").bfloat16()
    a = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    a[12] = math.nan
    a[35, 5] = math.inf
    c = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    h = device.stage_experts(w)
    device.gemm_grouped(h, a, M, torch.from_numpy(off).cuda(), M, K, N, c)
    device.sync()
    rows = set((~torch.isfinite(c)).any(1).nonzero().flatten().tolist())
    assert rows == {12, 35}
    device.release_weight(h)
    a = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    w[1] = math.nan
    h = device.stage_experts(w)
    device.gemm_grouped(h, a, M, torch.from_numpy(off).cuda(), M, K, N, c)
    device.sync()
    bad = (~torch.isfinite(c)).any(1).nonzero().flatten().tolist()
    assert bad == list(range(10, 30))
    device.release_weight(h)


def test_grouped_product_equals_one_product(device):
    """One expert over all rows is nebw_gemm's product: within a rounding."""
    M, K, N = 333, 384, 512
    g = gen(2)
    a = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    w = torch.randn(K, N, generator=g, device="cuda").bfloat16()
    bits = w.view(torch.int16).cpu().numpy().view(np.uint16)
    one, many = device.stage_weight(bits), device.stage_experts(bits[None])
    c1 = torch.empty(M, N, device="cuda")
    c2 = torch.empty(M, N, device="cuda")
    device.gemm(one, a, M, K, N, c1, c_dtype=0)
    device.gemm_grouped(many, a, M, torch.tensor([0, M], device="cuda").int(), M, K, N, c2,
                        c_dtype=0)
    device.sync()
    size = a.double().abs() @ w.double().abs()
    assert ((c1 - c2).abs().double() <= 4 * (K + 2) * U * size).all()
    device.release_weight(one)
    device.release_weight(many)


def test_grouped_product_without_the_pair_gemm(device, monkeypatch):
    """NEBW_GEMM_CTAS=1 takes nebw_gemm off CTA pairs, not the grouped product."""
    import nebw
    monkeypatch.setenv("NEBW_GEMM_CTAS", "1")
    other = nebw.Device(0, torch_stream=True)
    K, N, off = 128, 64, groups([3, 0, 40])
    w = torch.randn(3, K, N, generator=gen(18), device="cuda").bfloat16()
    a = torch.randn(43, K, generator=gen(19), device="cuda").bfloat16()
    c = torch.empty(43, N, dtype=torch.bfloat16, device="cuda")
    h = other.stage_experts(w)
    other.gemm_grouped(h, a, 43, torch.from_numpy(off).cuda(), 43, K, N, c)
    other.sync()
    assert_close(c, *grouped_reference(a, w, off, None, None, False, 0))
    other.close()


@pytest.mark.parametrize("source", ["numpy f32", "numpy bf16", "torch f32", "torch bf16", "cpu"])
def test_stage_experts_sources(device, source):
    """Weights from host or device memory, fp32 rounded to nearest even."""
    E, K, N = 3, 72, 64
    off = groups([4, 0, 9])
    w = torch.randn(E, K, N, generator=gen(3), device="cuda")
    wb = w.bfloat16()
    src = {"numpy f32": w.cpu().numpy(), "torch f32": w, "torch bf16": wb, "cpu": w.cpu(),
           "numpy bf16": wb.view(torch.int16).cpu().numpy().view(np.uint16)}[source]
    a = torch.randn(13, K, generator=gen(4), device="cuda").bfloat16()
    for gated in (False, True):
        h = device.stage_experts(src, gated=gated)
        c = torch.empty(13, N // 2 if gated else N, dtype=torch.bfloat16, device="cuda")
        device.gemm_grouped(h, a, 13, torch.from_numpy(off).cuda(), 13, K, N, c)
        device.sync()
        assert_close(c, *grouped_reference(a, wb, off, None, None, gated, 0))
        device.release_weight(h)


@pytest.mark.parametrize("off", [[0, 5, 3, 20], [0, 5, 10, 21], [-4, 5, 10, 20], [0, 30, 10, 20],
                                 [7, 2, 1, 0]])
def test_grouped_product_reports_bad_offsets(device, off):
    """Offsets that fall or leave the rows are reported; nothing outside C is written."""
    import nebw
    K = N = 64
    a = torch.randn(20, K, generator=gen(5), device="cuda").bfloat16()
    w = torch.randn(3, K, N, generator=gen(6), device="cuda").bfloat16()
    buf = torch.full((60, N), 7.0, dtype=torch.bfloat16, device="cuda")
    h = device.stage_experts(w)
    device.gemm_grouped(h, a, 20, torch.tensor(off, device="cuda").int(), 20, K, N, buf[20:40])
    with pytest.raises(nebw.NebwError, match="group"):
        device.sync()
    assert (buf[:20] == 7.0).all() and (buf[40:] == 7.0).all()
    device.sync()  # reported once
    device.release_weight(h)


def test_grouped_product_reports_bad_rows(device):
    """A row index outside A is reported and another row read in its place."""
    import nebw
    K = N = 64
    a = torch.randn(20, K, generator=gen(7), device="cuda").bfloat16()
    w = torch.randn(1, K, N, generator=gen(8), device="cuda").bfloat16()
    c = torch.empty(8, N, dtype=torch.bfloat16, device="cuda")
    h = device.stage_experts(w)
    off = groups([8])
    for bad in (20, -1, 2 ** 31 - 1):
        src = torch.arange(8, device="cuda").int()
        src[3] = bad
        device.gemm_grouped(h, a, 20, torch.from_numpy(off).cuda(), 8, K, N, c, row_src=src)
        with pytest.raises(nebw.NebwError, match="group"):
            device.sync()
        keep = [0, 1, 2, 4, 5, 6, 7]
        want, err = grouped_reference(a, w, off, torch.arange(8), None, False, 0)
        assert_close(c[keep], want[keep], err[keep])
    device.release_weight(h)


def test_grouped_refusals(device):
    import nebw
    a = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    c = torch.full((8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2, 64, 64, dtype=torch.bfloat16, device="cuda")
    off = torch.tensor([0, 4, 8], device="cuda").int()
    plain, gated = device.stage_experts(w), device.stage_experts(w, gated=True)

    def refused(word, fn, *args, **kw):
        with pytest.raises(nebw.NebwError, match=word) as e:
            fn(*args, **kw)
        assert e.value.code == 1

    g = device.gemm_grouped
    refused("unknown expert", g, plain + 1000, a, 8, off, 8, 64, 64, c)
    refused("does not match", g, plain, a, 8, off, 8, 128, 64, c)
    refused("does not match", g, plain, a, 8, off, 8, 64, 128, c)
    refused("rows", g, plain, a, 8, off, -1, 64, 64, c)
    refused("rows", g, plain, a, 8, off, 9, 64, 64, c.data_ptr())  # more groups than A has rows
    refused("empty A", g, plain, a, 0, off, 8, 64, 64, c, row_src=torch.zeros(8).int().cuda())
    for few in ((a, 9, off, 8, 64, 64, c), (a, 8, off, 9, 64, 64, c), (a, 8, off[:2], 8, 64, 64, c)):
        with pytest.raises(ValueError):  # fewer values than the call reads or writes
            g(plain, *few)
    with pytest.raises(ValueError):
        g(plain, a, 8, off, 8, 64, 64, c, row_src=off)
    with pytest.raises(ValueError):
        g(plain, a, 8, off, 8, 64, 64, c, bias=torch.zeros(64, device="cuda"))
    refused("activation", g, plain, a, 8, off, 8, 64, 64, c, act=3)
    refused("activation", g, gated, a, 8, off, 8, 64, 64, c, act=2)
    f = torch.zeros(8, 64, device="cuda")
    refused("bf16 output", g, plain, a, 8, off, 8, 64, 64, f, act=1, c_dtype=0)
    refused("bf16 output", g, gated, a, 8, off, 8, 64, 64, f, c_dtype=0)
    refused("output dtype", g, plain, a, 8, off, 8, 64, 64, c.data_ptr(), c_dtype=7)
    for bad in (a.float(), a.t(), a.cpu()):  # read as other numbers, or not at all
        with pytest.raises(TypeError):
            g(plain, bad, 8, off, 8, 64, 64, c)
    with pytest.raises(TypeError):
        g(plain, a, 8, off, 8, 64, 64, f)
    refused("null grouped", g, plain, None, 8, off, 8, 64, 64, c)
    refused("null grouped", g, plain, a, 8, None, 8, 64, 64, c)
    refused("aligned", g, plain, a.data_ptr() + 2, 7, off, 7, 64, 64, c)
    refused("aligned", g, plain, a, 8, off, 8, 64, 64, c.data_ptr() + 8)
    refused("expert weights", device.stage_experts, np.zeros((2, 56, 64), np.float32))
    refused("expert weights", device.stage_experts, np.zeros((2, 68, 64), np.float32))
    refused("expert weights", device.stage_experts, np.zeros((2, 64, 12), np.float32))
    refused("gated", device.stage_experts, np.zeros((2, 64, 96), np.float32), gated=True)
    refused("experts refused", device.stage_experts, np.zeros((513, 64, 8), np.float32))
    with pytest.raises(TypeError):
        device.stage_experts(np.zeros((2, 64, 64)))
    with pytest.raises(ValueError):  # not as it lies in memory
        device.stage_experts(torch.zeros(2, 64, 64, device="cuda").transpose(1, 2))
    g(plain, a, 8, off, 0, 64, 64, c)  # no rows: nothing to do
    device.sync()
    assert (c == 7.0).all()
    device.release_weight(plain)
    device.release_weight(gated)
    refused("unknown expert", g, plain, a, 8, off, 8, 64, 64, c)


def test_grouped_product_and_combine_past_32_bits(device):
    """An output of more than 2^31 elements, and the combine that reads it."""
    M, K, N = 270000, 64, 8192
    a = torch.randn(M, K, generator=gen(15), device="cuda").bfloat16()
    w = torch.randn(2, K, N, generator=gen(16), device="cuda").bfloat16()
    off = groups([M - 1000, 1000])
    h = device.stage_experts(w)
    c = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")  # 4.4 GB
    device.gemm_grouped(h, a, M, torch.from_numpy(off).cuda(), M, K, N, c)
    rows = 50
    dst = torch.stack([torch.arange(rows), M - 1 - torch.arange(rows)], 1).int().cuda()
    weights = torch.rand(rows, 2, generator=gen(17), device="cuda")
    out = torch.empty(rows, N, device="cuda")
    device.moe_combine(c, dst, weights, rows, 2, N, out)
    device.sync()
    at = torch.cat([torch.arange(300), torch.arange(M - 1300, M)]).cuda()
    want, err = grouped_reference(a[at], w, [0, 600, 1600], None, None, False, 0)
    assert_close(c[at], want, err)
    parts = c[dst.long()].double() * weights[:, :, None].double()
    assert_close(out, parts.sum(1), 3 * U * parts.abs().sum(1))
    device.release_weight(h)


def test_operands_off_their_values_boundaries_are_refused(device):
    """Addresses between two values are refused before a kernel reads there."""
    import nebw
    rows, E, k, H = 4, 8, 2, 64
    x = torch.zeros(rows, H, dtype=torch.bfloat16, device="cuda")
    it = torch.zeros(64, dtype=torch.int32, device="cuda")
    fl = torch.zeros(rows, H, device="cuda")
    inv, _ = nebw.rope_freqs(10000.0, H)
    rope = device.stage_rope(inv, 16)
    w = device.stage_experts(np.zeros((1, H, H), np.float32))
    a, p, f = x.data_ptr(), it.data_ptr(), fl.data_ptr()
    L, st = nebw.lib(), nebw.CUDA_STREAM_LEGACY
    side = nebw.Heads(a, a, H, H, 1)

    def swap(args, i, by):
        return [v + by if j == i else v for j, v in enumerate(args)]

    calls = [  # the call, its arguments, where the addresses are, and by how much they are off
        (L.nebw_packed_positions, [p, p, 1, 4, 4, p, st], (0, 1, 5), 2),
        (L.nebw_row_positions, [p, p, 1, 4, p, st], (0, 1, 4), 1),
        (L.nebw_rope, [side, None, nebw.BF16, rows, p, H, rope, 0, p, st], (4, 8), 2),
        (L.nebw_qk_norm_rope, [nebw.Heads(a, a, H, H, 1, 0, f), None, nebw.BF16, rows, p, H, 1,
                               1e-6, rope, 0, p, st], (4, 10), 2),
        (L.nebw_moe_route, [f, nebw.F32, E, rows, p, E, k, 0, 0, 1.0, p, f, p, p, p, p, 64 * 4,
                            st], (0, 4, 10, 11, 12, 13, 14, 15), 2),
        (L.nebw_gemm_grouped, [w, a, rows, p, p, rows, H, H, None, 0, f, nebw.BF16, st], (3, 4), 2),
        (L.nebw_moe_combine, [a, nebw.BF16, rows, p, f, rows, p, k, H, f, f, nebw.F32, st],
         (3, 4, 6, 9, 10), 2),
        (L.nebw_moe_combine, [a, nebw.BF16, rows, p, f, rows, p, k, H, None, a, nebw.BF16, st],
         (0, 10), 1),
    ]
    for call, args, where, by in calls:
        for i in where:
            assert call(device.h, *swap(args, i, by)) == 1, (call.__name__, i)
            assert "aligned" in L.nebw_last_error().decode(), (call.__name__, i)
    hnd = (nebw.C.c_uint64 * 1)()
    assert L.nebw_stage_experts(device.h, a + 1, nebw.BF16, 1, 64, 8, 0, st, hnd) == 1
    assert "aligned" in L.nebw_last_error().decode()
    device.sync()
    device.release_weight(rope)
    device.release_weight(w)


def test_results_over_what_is_still_read_are_refused(device):
    """Blocks run in no order: results may lie on their own operand, or beside
    everything that another block reads or writes, and nowhere between."""
    import nebw
    rows, hd = 5, 64
    buf = torch.zeros(40, 6 * hd, dtype=torch.bfloat16, device="cuda")
    inv, _ = nebw.rope_freqs(10000.0, hd)
    table = device.stage_rope(inv, 64)
    pos = torch.arange(40, device="cuda").int()

    def heads(at, n=1, out=None, rows=rows):
        v = [buf.flatten()[i:i + rows * 6 * hd].view(rows, 6 * hd)[:, :n * hd]
             for i in (at, at if out is None else out)]
        return nebw.Heads.of(v[0], n, out=v[1])

    wide = 6 * hd
    fine = [  # query, key (offsets of their first elements, heads, offsets of the results)
        (heads(0, 2), heads(2 * hd, 2)), (heads(0, 2, 4 * hd), heads(2 * hd, 2)),
        (heads(0, 2, wide * rows), heads(2 * hd, 2, wide * rows + 2 * hd)),
        (heads(wide, 3, 3 * hd), None), (heads(0, 3, wide * 2 + 3 * hd), None),
        (heads(wide * rows, 1, 0), heads(hd, 1)),
    ]
    bad = [
        (heads(0, 2, hd), None), (heads(hd, 2, 0), None), (heads(0, 2, wide), None),
        (heads(wide * 2, 2, 0), None), (heads(0, 1, wide - hd + 8), heads(0, 2, wide * 20)),
        (heads(0, 2), heads(0, 2)), (heads(0, 2), heads(hd, 2)),
        (heads(0, 2, wide * 10), heads(4 * hd, 2, wide * 10)),
        (heads(0, 2, 4 * hd), heads(4 * hd, 2, wide * 10)),
        (heads(2 * hd, 4, wide * 10 + 2 * hd), heads(0, 2, wide * 11 - 2 * hd)),
    ]
    for q, k in fine:
        device.rope(q, k, rows, hd, table, pos)
    for q, k in bad:
        for a, b in ((q, k), (k, q)):
            with pytest.raises(nebw.NebwError, match="overlap") as e:
                device.rope(a, b, rows, hd, table, pos)
            assert e.value.code == 1
    one = [nebw.Heads.of(buf[i:i + 1, :2 * hd], 2) for i in (0, 1)]
    device.rope(*one, 1, hd, table, pos)  # a row each
    with pytest.raises(nebw.NebwError, match="overlap"):
        device.rope(one[0], nebw.Heads.of(buf[:1, hd:3 * hd], 2), 1, hd, table, pos)
    device.release_weight(table)

    E, K, N, M = 1, 64, 64, 16
    w = device.stage_experts(np.zeros((E, K, N), np.float32))
    flat = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    off = torch.tensor([0, M], device="cuda").int()
    rows_of = lambda i, n: flat[i:i + n * K].view(n, K)  # noqa: E731
    device.gemm_grouped(w, rows_of(0, M), M, off, M, K, N, rows_of(M * K, M))
    for i in (0, 64, M * K - 64):
        with pytest.raises(nebw.NebwError, match="overlap"):
            device.gemm_grouped(w, rows_of(512, M), M, off, M, K, N, rows_of(512 + i, M))
        with pytest.raises(nebw.NebwError, match="overlap"):
            device.gemm_grouped(w, rows_of(512 + i, M), M, off, M, K, N, rows_of(512, M))
    device.release_weight(w)

    dst, wt = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.zeros(4, 1, device="cuda")
    y, f = rows_of(0, 8), torch.zeros(1024, device="cuda")
    device.moe_combine(y, dst, wt, 4, 1, K, rows_of(512, 4))
    for i in (0, 448):
        with pytest.raises(nebw.NebwError, match="overlap"):
            device.moe_combine(y, dst, wt, 4, 1, K, rows_of(i, 4))
    res = f[256:512].view(4, K)
    device.moe_combine(y, dst, wt, 4, 1, K, res, residual=res)
    r = Routing(1200, 8, 2)
    x = torch.zeros(1200, 8, device="cuda")
    given = [r.ids, r.weights, r.off, r.src, r.dst, r.ws]
    device.moe_route(x, 1200, 8, 2, *given)
    assert r.ws.numel()  # two kernels
    for i, t in enumerate(given):
        onto = x.flatten()[-t.numel():] if i == 1 else x.view(torch.int32).flatten()[-t.numel():]
        for j, other in ((None, onto), *((j, u) for j, u in enumerate(given) if j != i)):
            if j is not None:
                at = other.view(torch.float32 if i == 1 else torch.int32).flatten()
                if at.numel() < t.numel():
                    continue
                other = at[-t.numel():]
            new = list(given)
            new[i] = other.view(t.shape)
            with pytest.raises(nebw.NebwError, match="overlap"):
                device.moe_route(x, 1200, 8, 2, *new)
    for out in (f[192:448].view(4, K), f[260:516].view(4, K), res.view(torch.bfloat16).view(8, K)):
        with pytest.raises(nebw.NebwError, match="overlap"):
            device.moe_combine(y, dst, wt, 4, 1, K, out, residual=res)
    device.sync()


def test_whole_numbers_of_another_dtype_are_refused(device):
    """int64 indices (torch's default) would be read as other numbers, host
    memory not at all."""
    import nebw
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    inv, _ = nebw.rope_freqs(10000.0, 64)
    h = device.stage_rope(inv, 16)
    w = device.stage_experts(np.zeros((1, 64, 64), np.float32))
    with pytest.raises(TypeError):
        device.rope(nebw.Heads.of(x, 1), None, 4, 64, h, torch.arange(4, device="cuda"))
    with pytest.raises(TypeError):
        device.rope(nebw.Heads.of(x.cpu(), 1), None, 4, 64, h, torch.arange(4, device="cuda").int())
    with pytest.raises(TypeError):
        device.gemm_grouped(w, x, 4, torch.tensor([0, 4], device="cuda"), 4, 64, 64, x.clone())
    with pytest.raises(TypeError):  # every second value
        device.moe_combine(x, torch.zeros(4, 2, dtype=torch.int32, device="cuda")[:, :1],
                           torch.zeros(4, 1, device="cuda"), 4, 1, 64, x.clone())
    device.release_weight(h)
    device.release_weight(w)


# ---------------------------------------------------------------------------
# the combine
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("y_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,k,H", [(1, 1, 8), (1, 2, 768), (7, 2, 384), (100, 8, 1024),
                                      (33, 3, 520), (50, 4, 13), (9, 16, 2048), (1, 1, 1),
                                      (301, 2, 100)])
def test_combine_matches_64_bits(device, rows, k, H, y_dtype, out_dtype, residual):
    g = gen(rows + k + H)
    n = rows * k + 5
    y = torch.randn(n, H, generator=g, device="cuda").to(TYPES[y_dtype])
    dst = torch.randperm(n, generator=g, device="cuda")[:rows * k].reshape(rows, k).int()
    w = torch.rand(rows, k, generator=g, device="cuda")
    gone = torch.rand(rows, k, generator=g, device="cuda") < 0.2
    if rows > 2:
        gone[1] = True  # a row that went to no expert
    dst[gone] = -1
    w[gone] = math.nan  # not looked at
    res = torch.randn(rows, H, generator=g, device="cuda") if residual else None
    out = torch.full((rows + 1, H), 7.0, dtype=TYPES[out_dtype], device="cuda")
    device.moe_combine(y, dst, w, rows, k, H, out, residual=res)
    device.sync()
    parts = torch.where(gone[:, :, None], 0.0,
                        y[dst.clamp(min=0).long()].double() * w[:, :, None].double())
    want, size = parts.sum(1), parts.abs().sum(1)
    if residual:
        want, size = want + res.double(), size + res.double().abs()
    assert_close(out[:rows], want, (k + 1) * U * size)
    assert (out[rows:] == 7.0).all()


def test_combine_in_place_residual_live_rows_and_bad_places(device):
    import nebw
    rows, k, H = 37, 2, 256
    g = gen(11)
    y = torch.randn(rows * k, H, generator=g, device="cuda").bfloat16()
    dst = torch.randperm(rows * k, generator=g, device="cuda").reshape(rows, k).int()
    w = torch.rand(rows, k, generator=g, device="cuda")
    x = torch.randn(rows, H, generator=g, device="cuda")
    parts = y[dst.long()].double() * w[:, :, None].double()
    want = x.double() + parts.sum(1)
    for live in (0, 1, 20, 37, 100, -5):
        out = x.clone()
        n = torch.tensor([live], dtype=torch.int32, device="cuda")
        device.moe_combine(y, dst, w, rows, k, H, out, residual=out, rows_dev=n)
        device.sync()
        live = max(0, min(live, rows))
        assert torch.equal(out[live:], x[live:])
        size = parts.abs().sum(1) + x.double().abs()
        assert_close(out[:live], want[:live], 3 * U * size[:live])
    bad = dst.clone()
    bad[5, 1] = rows * k
    out = torch.empty(rows, H, device="cuda")
    device.moe_combine(y, bad, w, rows, k, H, out, residual=x)
    with pytest.raises(nebw.NebwError, match="group"):
        device.sync()
    want[5] = x[5].double() + parts[5, 0]
    assert_close(out, want, 3 * U * (parts.abs().sum(1) + x.double().abs()))


def test_combine_unaligned_rows(device):
    """Buffers off a 16-byte boundary give the aligned call's bits."""
    rows, k, H = 21, 2, 64
    g = gen(12)
    y = torch.randn(rows * k, H, generator=g, device="cuda").bfloat16()
    dst = torch.randperm(rows * k, generator=g, device="cuda").reshape(rows, k).int()
    w = torch.rand(rows, k, generator=g, device="cuda")
    out = torch.empty(rows, H, dtype=torch.bfloat16, device="cuda")
    device.moe_combine(y, dst, w, rows, k, H, out)
    ybuf = torch.empty(rows * k * H + 1, dtype=torch.bfloat16, device="cuda")
    y2 = ybuf[1:].view(rows * k, H)
    y2.copy_(y)
    obuf = torch.empty(rows * H + 3, dtype=torch.bfloat16, device="cuda")
    out2 = obuf[3:].view(rows, H)
    device.moe_combine(y2, dst, w, rows, k, H, out2)
    device.sync()
    assert torch.equal(out, out2)


def test_combine_refusals(device):
    import nebw
    y = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    dst = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, 2, device="cuda")
    out = torch.full((4, 64), 7.0, device="cuda")

    def refused(word, *args, **kw):
        with pytest.raises(nebw.NebwError, match=word) as e:
            device.moe_combine(*args, **kw)
        assert e.value.code == 1

    refused("top_k", y, dst, w, 4, 0, 64, out)
    many = torch.zeros(4, 17, device="cuda")
    refused("top_k", y, many.int(), many, 4, 17, 64, out)
    for few in ((y, dst, w, 5, 2, 64, out), (y, dst, w, 4, 2, 72, out), (y, dst, w[:3], 4, 2, 64, out)):
        with pytest.raises(ValueError):  # fewer values than the call reads or writes
            device.moe_combine(*few)
    refused("width", y, dst, w, 4, 2, 0, out)
    refused("rows", y, dst, w, -1, 2, 64, out)
    refused("null combine", y, None, w, 4, 2, 64, out)
    with pytest.raises(TypeError):
        device.moe_combine(y.half(), dst, w, 4, 2, 64, out)
    device.moe_combine(y, dst, w, 0, 2, 64, out)
    device.sync()
    assert (out == 7.0).all()
    # no expert's rows at all, and no place that would need one
    device.moe_combine(y[:0].clone(), torch.full_like(dst, -1), w, 4, 2, 64, out)
    device.sync()
    assert (out == 0.0).all()


# ---------------------------------------------------------------------------
# the operators together, as a layer uses them
# ---------------------------------------------------------------------------

class Layer:
    """One rotary expert layer's buffers and weights, post-norm:
    Q|K|V product, head norms with rotation, attention, output product,
    LayerNorm; router product, routing, the experts' two products, combine,
    LayerNorm."""

    H, HEADS, E, K, F = 256, 4, 8, 2, 128

    def __init__(self, device, T, seed=20):
        import nebw
        self.dev, self.T = device, T
        g = gen(seed)
        H, E, F, k = self.H, self.E, self.F, self.K

        def randn(*s, by=1.0):
            return by * torch.randn(*s, generator=g, device="cuda")

        self.w = dict(qkv=randn(H, 3 * H, by=0.06), ao=randn(H, H, by=0.06),
                      router=randn(H, E, by=0.1))
        self.up, self.down = randn(E, H, 2 * F, by=0.06), randn(E, F, H, by=0.09)
        self.stage = {n: device.stage_weight(v.cpu().numpy()) for n, v in self.w.items()}
        self.h_up = device.stage_experts(self.up, gated=True)
        self.h_down = device.stage_experts(self.down)
        self.inv, _ = nebw.rope_freqs(10000.0, 64)
        self.rope = device.stage_rope(self.inv, 512)
        self.gam = [1 + randn(64, by=0.1) for _ in range(2)]
        # Q's 1/sqrt(head_dim) lies in its norm's weight
        self.gam[0] = self.gam[0] / 8.0
        self.ln = [torch.ones(H, device="cuda"), torch.zeros(H, device="cuda")]
        bf = dict(dtype=torch.bfloat16, device="cuda")
        it = dict(dtype=torch.int32, device="cuda")
        self.qkv, self.ctx = torch.zeros(T, 3 * H, **bf), torch.zeros(T, H, **bf)
        self.y, self.a = torch.zeros(T, H, **bf), torch.zeros(T, H, **bf)
        self.logits = torch.zeros(T, E, device="cuda")
        self.ids, self.dst = torch.zeros(T, k, **it), torch.zeros(T, k, **it)
        self.weights = torch.zeros(T, k, device="cuda")
        self.off, self.src = torch.zeros(E + 1, **it), torch.zeros(T * k, **it)
        self.ws = torch.zeros(nebw.moe_route_workspace(T, E, k), dtype=torch.uint8, device="cuda")
        self.hid, self.yk = torch.zeros(T * k, F, **bf), torch.zeros(T * k, H, **bf)
        self.heads = [nebw.Heads.of(self.qkv[:, i * H:(i + 1) * H], self.HEADS, gamma=self.gam[i])
                      for i in range(2)]

    def run(self, x, pos, off, lens, live=None):
        import nebw
        d, T, H, E, k, F = self.dev, self.T, self.H, self.E, self.K, self.F
        B, S = len(lens), 128
        d.gemm(self.stage["qkv"], self.a, T, H, 3 * H, self.qkv)
        d.qk_norm_rope(*self.heads, T, 64, rope=self.rope, pos=pos, rows_dev=live)
        d.attention(self.qkv, T, off, lens, B, S, self.HEADS, 64, self.ctx)
        d.gemm(self.stage["ao"], self.ctx, T, H, H, self.y)
        d.layernorm(x, *self.ln, T, H, y=self.y, a_bf16=self.a)
        d.gemm(self.stage["router"], self.a, T, H, E, self.logits, c_dtype=nebw.F32)
        d.moe_route(self.logits, T, E, k, self.ids, self.weights, self.off, self.src, self.dst,
                    self.ws, renorm=True, rows_dev=live)
        d.gemm_grouped(self.h_up, self.a, T, self.off, T * k, H, 2 * F, self.hid,
                       row_src=self.src, act=nebw.GATE_SILU)
        d.gemm_grouped(self.h_down, self.hid, T * k, self.off, T * k, F, H, self.yk)
        d.moe_combine(self.yk, self.dst, self.weights, T, k, H, self.y, rows_dev=live)
        d.layernorm(x, *self.ln, T, H, y=self.y, a_bf16=self.a)

    def close(self):
        for h in list(self.stage.values()) + [self.h_up, self.h_down, self.rope]:
            self.dev.release_weight(h)

    def reference(self, x, pos, lens):
        """The layer in 64 bits on bf16 weights (fp32 activations unrounded)."""
        H, n = self.H, self.HEADS
        bf = lambda t: t.bfloat16().double()  # noqa: E731
        norm = lambda t: torch.nn.functional.layer_norm(t, (H,), eps=1e-12)  # noqa: E731
        x = x.double()
        qkv = bf(x) @ bf(self.w["qkv"])
        side = [heads_reference(qkv[:, i * H:(i + 1) * H], n, 64, self.inv, 1.0, pos, False, 1,
                                self.gam[i], None, 1e-6)[0].view(-1, n, 64) for i in range(2)]
        v = qkv[:, 2 * H:].view(-1, n, 64)
        ctx, at = [], 0
        for length in lens:
            s = slice(at, at + length)
            p = torch.softmax(torch.einsum("qhd,khd->hqk", side[0][s], side[1][s]), -1)
            ctx.append(torch.einsum("hqk,khd->qhd", p, v[s]).reshape(length, H))
            at += length
        x = norm(x + torch.cat(ctx) @ bf(self.w["ao"]))
        logits = x @ bf(self.w["router"])
        best = logits.sort(dim=1, descending=True, stable=True)
        p = torch.softmax(best.values[:, :self.K], 1)
        out = torch.zeros_like(x)
        for j in range(self.K):
            e = best.indices[:, j]
            ug = torch.einsum("th,thf->tf", x, bf(self.up)[e])
            u, gate = ug.chunk(2, 1)
            out += p[:, j:j + 1] * torch.einsum("tf,tfh->th", u * gate * torch.sigmoid(gate),
                                                bf(self.down)[e])
        # how clear each row's choice of experts is
        clear = best.values[:, self.K - 1] - best.values[:, self.K]
        return norm(x + out), clear


def test_layer_of_the_operators_together(device):
    lens = [100, 1, 37, 128, 5]
    T = sum(lens)
    layer = Layer(device, T)
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    n, off = torch.empty_like(lens_d), torch.empty(len(lens) + 1, dtype=torch.int32, device="cuda")
    device.pack_offsets(lens_d, len(lens), 128, n, off)
    pos = torch.empty(T, dtype=torch.int32, device="cuda")
    device.row_positions(off, n, len(lens), 128, pos)
    x0 = torch.randn(T, layer.H, generator=gen(21), device="cuda")
    x = x0.clone()
    layer.a.copy_(x0)
    layer.run(x, pos, off, n)
    device.sync()
    want, clear = layer.reference(x0, pos, lens)
    # rows whose second and third expert are nearly even may go either way:
    # the logits come from rows rounded to bf16 (2^-8 of about 1, 256 terms of
    # 0.1: a standard deviation of 0.004)
    sure = clear > 0.05
    assert sure.sum() > 0.8 * T
    diff = (x.double() - want)[sure]
    # activations are rounded to bf16 seven times on the way, each 2^-9 of
    # unit-sized rows in the mean square
    assert diff.square().mean().sqrt() <= 7 * 2.0 ** -9 and diff.abs().max() <= 0.1
    # the same layer replayed from one graph, on other inputs and a live count
    # that the capture did not see
    live = torch.tensor([T], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer.a.copy_(x0)
        x.copy_(x0)
        layer.run(x, pos, off, n, live)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.run(x, pos, off, n, live)
    torch.cuda.synchronize()
    x1 = torch.randn(T, layer.H, generator=gen(22), device="cuda")
    for start, count in ((x0, T), (x1, T), (x1, 138)):
        live.fill_(count)
        x.copy_(start)
        layer.a.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        got = x[:count].clone()
        x.copy_(start)
        layer.a.copy_(start)
        layer.run(x, pos, off, n)
        device.sync()
        # a live count of whole sequences drops the rows behind, no others
        assert torch.equal(got, x[:count])
    layer.close()


def test_operators_on_another_stream(device):
    """Calls on a stream of the caller's own follow that stream's work."""
    import nebw
    rows, E, k, H = 2000, 16, 2, 256
    side = torch.cuda.Stream()
    x = torch.randn(rows, E, generator=gen(30), device="cuda")
    w = torch.randn(E, H, H, generator=gen(31), device="cuda").bfloat16()
    a = torch.randn(rows, H, generator=gen(32), device="cuda").bfloat16()
    h = device.stage_experts(w)
    torch.cuda.synchronize()
    outs = []
    for stream in (None, side):
        with torch.cuda.stream(stream or torch.cuda.current_stream()):
            r = Routing(rows, E, k)
            yk = torch.empty(rows * k, H, dtype=torch.bfloat16, device="cuda")
            out = torch.empty(rows, H, device="cuda")
            late = x * 2 - x  # written on this stream just before it is read
            r.run(device, late, renorm=True)
            device.gemm_grouped(h, a, rows, r.off, rows * k, H, H, yk, row_src=r.src)
            device.moe_combine(yk, r.dst, r.weights, rows, k, H, out)
        torch.cuda.synchronize()
        outs.append(out)
    assert torch.equal(*outs)
    device.release_weight(h)


def test_two_threads_on_two_streams_at_once(device):
    """Two threads with a stream and a workspace each share a handle and its
    staged weights."""
    import threading
    rows, E, k, H, N = 700, 16, 2, 256, 512
    w = torch.randn(E, H, N, generator=gen(41), device="cuda").bfloat16()
    h = device.stage_experts(w)
    xs = [torch.randn(rows, E, generator=gen(42 + i), device="cuda") for i in range(2)]
    a = torch.randn(rows, H, generator=gen(44), device="cuda").bfloat16()
    rs = [Routing(rows, E, k) for _ in range(4)]
    ys = [torch.empty(rows * k, N, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    outs = [torch.empty(rows, N, device="cuda") for _ in range(4)]

    def run(i, slot, stream=None):
        r = rs[slot]
        device.moe_route(xs[i], rows, E, k, r.ids, r.weights, r.off, r.src, r.dst, r.ws,
                         renorm=True, stream=stream)
        device.gemm_grouped(h, a, rows, r.off, rows * k, H, N, ys[slot], row_src=r.src,
                            stream=stream)
        device.moe_combine(ys[slot], r.dst, r.weights, rows, k, N, outs[slot], stream=stream)

    for i in range(2):
        run(i, 2 + i)
    torch.cuda.synchronize()
    errors = []

    def work(i, stream):
        try:
            for _ in range(20):
                run(i, i, stream)
            stream.synchronize()
        except Exception as e:  # pragma: no cover - the assertion below reports it
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i, torch.cuda.Stream())) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    device.sync()
    assert not errors
    for i in range(2):
        assert torch.equal(outs[i], outs[2 + i]) and torch.equal(rs[i].off, rs[2 + i].off)
    device.release_weight(h)


def test_staging_beside_running_operators(device):
    """One thread stages and releases tables and expert weights while two others
    look their own up: each has what it staged."""
    import threading

    import nebw
    rows, E, H, N, hd = 200, 4, 128, 128, 64
    w = torch.randn(E, H, N, generator=gen(51), device="cuda").bfloat16()
    a = torch.randn(rows, H, generator=gen(52), device="cuda").bfloat16()
    off = torch.from_numpy(groups([50, 0, 100, 50])).cuda()
    x = torch.randn(rows, 2 * hd, generator=gen(53), device="cuda").bfloat16()
    pos = torch.arange(rows, device="cuda").int()
    inv, _ = nebw.rope_freqs(10000.0, hd)
    table, experts = device.stage_rope(inv, rows), device.stage_experts(w)
    outs = [[torch.empty(rows, N, dtype=torch.bfloat16, device="cuda"), torch.empty_like(x)]
            for _ in range(3)]
    sides = [nebw.Heads.of(x, 2, out=o[1]) for o in outs]

    def run(i, stream=None):
        device.gemm_grouped(experts, a, rows, off, rows, H, N, outs[i][0], stream=stream)
        device.rope(sides[i], None, rows, hd, table, pos, stream=stream)

    run(2)
    torch.cuda.synchronize()
    stop, errors, seen = threading.Event(), [], set()

    def work(i, stream):
        try:
            for _ in range(400):
                run(i, stream)
            stream.synchronize()
        except Exception as e:  # pragma: no cover - the assertion below reports it
            errors.append(e)

    def stage():
        try:
            while not stop.is_set():
                new = [device.stage_rope(inv, 64) for _ in range(3)]
                new.append(device.stage_experts(np.zeros((1, 64, 64), np.float32)))
                seen.update(new)
                for h in new:
                    device.release_weight(h)
        except Exception as e:  # pragma: no cover
            errors.append(e)

    workers = [threading.Thread(target=work, args=(i, torch.cuda.Stream())) for i in range(2)]
    stager = threading.Thread(target=stage)
    for t in workers + [stager]:
        t.start()
    for t in workers:
        t.join()
    stop.set()
    stager.join()
    torch.cuda.synchronize()
    device.sync()
    assert not errors and seen and not seen & {table, experts}
    for i in range(2):
        assert torch.equal(outs[i][0], outs[2][0]) and torch.equal(outs[i][1], outs[2][1])
    device.release_weight(table)
    device.release_weight(experts)


FIRST_CALLS = """
import sys
import numpy as np, torch
sys.path[:0] = sys.argv[1:2]
import nebw
d = nebw.Device(0, torch_stream=True)
rows, E, k, H = 300, 256, 8, 128
g = torch.Generator(device="cuda").manual_seed(1)
logits = torch.randn(rows, E, generator=g, device="cuda")
a = torch.randn(rows, H, generator=g, device="cuda").bfloat16()
x = torch.randn(rows, 2 * H, generator=g, device="cuda").bfloat16()
gamma = torch.ones(64, device="cuda")
pos = torch.arange(rows, device="cuda").int()
w = d.stage_experts((torch.randn(E, H, H, generator=g, device="cuda") / 12).bfloat16())
table = d.stage_rope(nebw.rope_freqs(10000.0, 64)[0], rows)
it = dict(dtype=torch.int32, device="cuda")

def buffers():
    ws = torch.empty(nebw.moe_route_workspace(rows, E, k), dtype=torch.uint8, device="cuda")
    return (torch.zeros(rows, k, **it), torch.zeros(rows, k, device="cuda"), torch.zeros(E + 1, **it),
            torch.zeros(rows * k, **it), torch.zeros(rows, k, **it), ws,
            torch.zeros(rows * k, H, dtype=torch.bfloat16, device="cuda"),
            torch.zeros(rows, H, device="cuda"), torch.zeros_like(x))

def run(ids, weights, off, src, dst, ws, y, out, turned, n):
    d.moe_route(logits, n, E, k, ids, weights, off, src, dst, ws, renorm=True)
    d.gemm_grouped(w, a, rows, off, rows * k, H, H, y, row_src=src)
    d.moe_combine(y, dst, weights, n, k, H, out)
    d.qk_norm_rope(nebw.Heads.of(x, 4, out=turned, gamma=gamma), None, rows, 64, rope=table, pos=pos)

for n in (rows, 20):  # two routing kernels, and one
    one, two = buffers(), buffers()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        run(*one, n)
    graph.replay()
    run(*two, n)
    d.sync()
    assert all(torch.equal(s, t) for s, t in zip(one[:5] + one[6:], two[:5] + two[6:]))
    assert (one[7][:n] != 0).any()
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture(device):
    """The operators' kernels are made ready by the first call that needs them:
    that call may be one that a graph captures."""
    import subprocess
    import sys

    from conftest import PKG
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS, str(PKG)], capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stderr[-2000:]
