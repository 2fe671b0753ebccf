"""Host side of the rotary and expert operators (CPU, no device): the rotary
frequency sets against their formulas, the workspace sizes and the refusals
that need no GPU."""

import math

import numpy as np
import pytest


@pytest.mark.parametrize("n", [1, 2, 16, 32, 128])
@pytest.mark.parametrize("theta", [1000.0, 160000.0])
def test_rope_freqs_plain_linear_ntk(n, theta):
    import nebw
    i = np.arange(n)
    # a few roundings of pow in double
    tol = dict(rtol=1e-13, atol=0)
    inv, scale = nebw.rope_freqs(theta, 2 * n)
    assert scale == 1.0
    np.testing.assert_allclose(inv, theta ** (-i / n), **tol)
    inv, scale = nebw.rope_freqs(theta, 2 * n, "linear", factor=8.0)
    assert scale == 1.0
    np.testing.assert_allclose(inv, theta ** (-i / n) / 8.0, **tol)
    inv, scale = nebw.rope_freqs(theta, 2 * n, "ntk", factor=8.0)
    assert scale == 1.0
    np.testing.assert_allclose(inv[0], 1.0, **tol)
    if n > 1:  # the slowest frequency is the linear one, the fastest is kept
        np.testing.assert_allclose(inv[-1], theta ** (-(n - 1) / n) / 8.0, rtol=1e-12)


def test_rope_freqs_yarn_and_bands():
    import nebw
    n, theta, length, factor = 64, 10000.0, 4096, 16.0
    plain = theta ** (-np.arange(n) / n)
    turns = length * plain / (2 * math.pi)
    inv, scale = nebw.rope_freqs(theta, 2 * n, "yarn", factor=factor, orig_len=length)
    assert scale == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)
    ratio = plain / inv
    # a few roundings of pow in double
    np.testing.assert_allclose(ratio[turns > 40], 1.0, rtol=1e-13)      # fast ones are kept
    np.testing.assert_allclose(ratio[turns < 0.9], factor, rtol=1e-12)  # slow ones are divided
    assert np.all(np.diff(ratio) >= -1e-12)            # and between them it only grows
    assert nebw.rope_freqs(theta, 2 * n, "yarn", factor, length, attn_scale=1.5)[1] == 1.5
    inv, scale = nebw.rope_freqs(theta, 2 * n, "bands", factor=factor, orig_len=length)
    assert scale == 1.0
    ratio = plain / inv
    np.testing.assert_allclose(ratio[turns >= 4.0], 1.0, rtol=1e-13)
    np.testing.assert_allclose(ratio[turns <= 1.0], factor, rtol=1e-12)
    mid = (turns > 1.0) & (turns < 4.0)
    keep = (turns[mid] - 1.0) / 3.0
    np.testing.assert_allclose(inv[mid], plain[mid] * (keep + (1 - keep) / factor), rtol=1e-12)
    inv, _ = nebw.rope_freqs(theta, 2 * n, "bands", factor, length, fast=2.0, slow=0.5)
    np.testing.assert_allclose((plain / inv)[turns >= 2.0], 1.0, rtol=1e-13)


@pytest.mark.parametrize("theta,rot_dim,length,factor,fast,slow", [
    (10000.0, 128, 4096, 16.0, 0, 0),
    # the index that turns once lies past the last frequency
    (1000.0, 32, 4096, 8.0, 0, 0), (1000.0, 64, 8192, 8.0, 0, 0), (10000.0, 64, 131072, 4.0, 0, 0),
    (1000.0, 12, 4096, 2.0, 0, 0), (500000.0, 128, 8192, 8.0, 24.0, 0.25),
    # past rot_dim - 1, where it is bounded; every frequency turns fast
    (100.0, 16, 1 << 20, 8.0, 0, 0), (100.0, 16, 1 << 30, 8.0, 0, 0), (10000.0, 2, 4096, 4.0, 0, 0),
])
def test_rope_freqs_yarn_ramp(theta, rot_dim, length, factor, fast, slow):
    """Every frequency against the definition: the indices of the two turn
    counts, rounded outwards and held within [0, rot_dim - 1], a linear ramp
    between them, and the frequencies blended by it."""
    import nebw

    def index(turns):
        return rot_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low = max(math.floor(index(fast or 32)), 0)
    high = min(math.ceil(index(slow or 1)), rot_dim - 1)
    inv, _ = nebw.rope_freqs(theta, rot_dim, "yarn", factor, length, fast, slow)
    assert len(inv) == rot_dim // 2
    for i, got in enumerate(inv):
        plain = theta ** (-2.0 * i / rot_dim)
        ramp = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
        # a few roundings of pow and log in double
        assert got == pytest.approx(plain / factor * ramp + plain * (1 - ramp), rel=1e-12), i
        # and what the definition says of it in words
        if length * plain / (2 * math.pi) > 2.0 * (fast or 32):
            assert got == pytest.approx(plain, rel=1e-12)


def test_rope_freqs_yarn_where_no_frequency_turns():
    """A trained length in which not even the first frequency turns `slow`
    times: all of them are divided."""
    import nebw
    n, theta, length, factor = 32, 10000.0, 4, 8.0
    plain = theta ** (-np.arange(n) / n)
    assert (length * plain / (2 * math.pi) < 1.0).all()
    inv, _ = nebw.rope_freqs(theta, 2 * n, "yarn", factor, length, fast=32.0, slow=2.0)
    np.testing.assert_allclose(plain / inv, factor, rtol=1e-12)


@pytest.mark.parametrize("args,word", [
    ((10000.0, 7), "rotary width"),
    ((10000.0, 0), "rotary width"),
    ((10000.0, 258), "rotary width"),
    ((1.0, 64), "rotary base"),
    ((float("inf"), 64), "rotary base"),
    ((float("nan"), 64), "rotary base"),
    ((10000.0, 64, "linear", 0.5), "factor"),
    ((10000.0, 64, "ntk", float("nan")), "factor"),
    ((10000.0, 64, "yarn", 4.0), "trained length"),
    ((10000.0, 64, "bands", 4.0, 4096, 1.0, 2.0), "bounds"),
])
def test_rope_freqs_refusals(args, word):
    import nebw
    with pytest.raises(nebw.NebwError, match=word) as e:
        nebw.rope_freqs(*args)
    assert e.value.code == 1


def test_rope_freqs_null_outputs_and_unknown_kind():
    import ctypes as C

    import nebw
    L = nebw.lib()
    assert L.nebw_rope_freqs(10000.0, 64, None, None, None) == 1
    inv, scale = (C.c_double * 32)(), C.c_double()
    s = nebw.RopeScaling(9, 0, 4096, 2.0, 0, 0, 0)
    assert L.nebw_rope_freqs(10000.0, 64, C.byref(s), inv, C.byref(scale)) == 1
    assert "scaling 9" in L.nebw_last_error().decode()
    assert L.nebw_rope_freqs(10000.0, 64, None, inv, C.byref(scale)) == 0  # NULL: plain
    assert inv[0] == 1.0 and scale.value == 1.0


def test_route_workspace():
    import nebw
    assert nebw.moe_route_workspace(0, 8, 2) == 0
    small, big = nebw.moe_route_workspace(1, 8, 2), nebw.moe_route_workspace(131072, 256, 8)
    assert 0 <= small <= big <= 16 << 20
    for rows, experts, k in [(1, 0, 1), (1, 513, 1), (1, 8, 0), (1, 8, 17), (1, 4, 5), (-1, 8, 2),
                             (1 << 30, 8, 2), (1 << 62, 8, 4)]:
        with pytest.raises(nebw.NebwError):
            nebw.moe_route_workspace(rows, experts, k)


def test_a_library_of_an_earlier_build_is_refused(tmp_path, monkeypatch):
    """One that has the version but not what was added since is refused when it
    is loaded."""
    import re
    import shutil
    import subprocess

    import nebw
    text = nebw.HEADER_PATH.read_text()
    here = tuple(int(re.search(rf"#define NEBW_ABI_{n} (\d+)", text)[1])
                 for n in ("VERSION", "REVISION"))
    assert here == nebw.ABI == (nebw.lib().nebw_abi_version(), nebw.lib().nebw_abi_revision())
    cc = shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    src = "int nebw_abi_version(void) { return %d; }"
    newer = src + " int nebw_abi_revision(void) { return %d; }"
    for i, text in enumerate((src % here[0], newer % (here[0], here[1] - 1),
                              newer % (here[0] + 1, here[1]))):
        (tmp_path / f"{i}.c").write_text(text)
        out = tmp_path / f"lib{i}.so"
        subprocess.run([cc, "-shared", "-fPIC", "-o", out, tmp_path / f"{i}.c"], check=True)
        monkeypatch.setattr(nebw, "_lib", None)
        monkeypatch.setattr(nebw, "LIB_PATH", out)
        with pytest.raises(nebw.NebwError, match="another build"):
            nebw.lib()


def test_null_device_is_refused_by_name():
    import nebw
    L = nebw.lib()
    calls = {
        "nebw_stage_rope": (None, None, 1, 1, 1.0, None),
        "nebw_row_positions": (None,) * 3 + (1, 1, None, None),
        "nebw_rope": (None, None, None, 1, 1, None, 64, 1, 0, None, None),
        "nebw_qk_norm_rope": (None, None, None, 1, 1, None, 64, 1, 1e-6, 0, 0, None, None),
        "nebw_stage_experts": (None, None, 0, 1, 64, 64, 0, None, None),
        "nebw_moe_route": (None, None, 0, 8, 1, None, 8, 2, 0, 0, 1.0) + (None,) * 6 + (0, None),
        "nebw_gemm_grouped": (None, 1, None, 1, None, None, 1, 64, 64, None, 0, None, 1, None),
        "nebw_moe_combine": (None, None, 1, 1, None, None, 1, None, 2, 64, None, None, 1, None),
    }
    for name, args in calls.items():
        assert getattr(L, name)(*args) == 1, name
        assert "null device handle" in L.nebw_last_error().decode(), name


def test_released_experts_are_forgotten(monkeypatch):
    """What the handle's object knows of an expert weight goes with it."""
    import nebw

    class Lib:
        rc = 0

        def nebw_release_weight(self, h, handle):
            return self.rc

        def nebw_last_error(self):
            return b"unknown weight handle"

    stub = Lib()
    monkeypatch.setattr(nebw, "lib", lambda: stub)
    d = nebw.Device.__new__(nebw.Device)
    d.h, d.index, d._experts = None, 0, {3: (2, 64, 64, 64), 4: (2, 64, 64, 64)}
    d.release_weight(3)
    assert list(d._experts) == [4]
    d.release_weight(9)  # of another kind
    stub.rc = 1
    with pytest.raises(nebw.NebwError):
        d.release_weight(4)
    assert list(d._experts) == [4]
    stub.rc = 0
    d.release_weight(4)


def test_positions_say_how_many_they_are():
    """An address alone does not: nothing may be written without a bound."""
    import nebw
    L = nebw.lib()
    assert L.nebw_packed_positions(None, None, None, 1, 1, 1, None, None) == 1
    assert "null device handle" in L.nebw_last_error().decode()
    d = nebw.Device.__new__(nebw.Device)
    d.h, d.index = None, 0
    for nowhere in (64, None):
        with pytest.raises(ValueError):
            d.row_positions(64, 64, 1, 8, nowhere)


def test_heads_of_refuses_what_it_cannot_describe():
    torch = pytest.importorskip("torch")
    import nebw
    x = torch.zeros(4, 96)
    h = nebw.Heads.of(x[:, 32:], 2)
    assert (h.x, h.out, h.stride, h.heads) == (x.data_ptr() + 128, x.data_ptr() + 128, 96, 2)
    for bad in (x.t(), x[:, ::2], x.reshape(2, 2, 96)):
        with pytest.raises(ValueError):
            nebw.Heads.of(bad, 2)
    with pytest.raises(ValueError):
        nebw.Heads.of(x, 5)
    with pytest.raises(ValueError):
        nebw.Heads.of(x, 2, out=torch.zeros(4, 96, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        nebw.Heads.of(x, 2, gamma=torch.zeros(96))
    with pytest.raises(TypeError):
        nebw.Heads.of(x.double(), 2)


@pytest.fixture
def host_calls(monkeypatch):
    """A handle whose checks take host tensors, and the library calls that pass
    them (each answered with success)."""
    torch = pytest.importorskip("torch")
    import nebw

    class Lib:
        calls = []

        def __getattr__(self, name):
            return lambda *args: self.calls.append((name, args)) or 0

    stub = Lib()
    stub.calls = []
    monkeypatch.setattr(nebw, "lib", lambda: stub)
    d = nebw.Device.__new__(nebw.Device)
    # a host tensor's device number
    d.h, d.index, d._raw_stream, d.torch_stream = None, torch.zeros(1).get_device(), None, False
    d._experts = {}
    return d, stub.calls


def test_rows_of_another_width_are_refused(host_calls):
    """Rows wider than the call says would be read, or written, at the wrong
    places; other shapes with as many values a row are fine."""
    torch = pytest.importorskip("torch")
    import nebw
    d, calls = host_calls
    bf, i32 = torch.bfloat16, torch.int32
    dst, w = torch.zeros(4, 2, dtype=i32), torch.zeros(4, 2)

    def combine(y=torch.zeros(8, 64, dtype=bf), dst=dst, w=w, out=torch.zeros(4, 64), **kw):
        d.moe_combine(y, dst, w, 4, 2, 64, out, **kw)

    combine()
    assert calls[-1][1][3] == 8
    combine(y=torch.zeros(2, 8, 64, dtype=bf), dst=dst.flatten(), w=w.flatten(),
            out=torch.zeros(5 * 64), residual=torch.zeros(1, 4, 64))
    assert calls[-1][1][3] == 16  # all of its rows
    for bad in (dict(y=torch.zeros(8, 96, dtype=bf)), dict(out=torch.zeros(4, 128)),
                dict(residual=torch.zeros(4, 65)), dict(dst=torch.zeros(4, 3, dtype=i32)),
                dict(w=torch.zeros(4, 4))):
        with pytest.raises(ValueError):
            combine(**bad)
    d._experts[7] = (2, 64, 128, 64)  # gated

    def grouped(a=torch.zeros(4, 64, dtype=bf), out=torch.zeros(4, 64, dtype=bf), bias=None):
        d.gemm_grouped(7, a, 4, torch.zeros(3, dtype=i32), 4, 64, 128, out, bias=bias)

    grouped()
    grouped(torch.zeros(2, 3, 64, dtype=bf), torch.zeros(500, dtype=bf), torch.zeros(2, 128))
    for bad in (dict(a=torch.zeros(4, 72, dtype=bf)), dict(out=torch.zeros(4, 128, dtype=bf)),
                dict(bias=torch.zeros(2, 192))):
        with pytest.raises(ValueError):
            grouped(**bad)

    def route(ids=dst, w=w, dst=dst):
        d.moe_route(torch.zeros(4, 8), 4, 8, 2, ids, w, torch.zeros(9, dtype=i32),
                    torch.zeros(8, dtype=i32), dst, torch.zeros(0))

    route()
    route(torch.zeros(9, 2, dtype=i32), torch.zeros(20), torch.zeros(4, 2, dtype=i32))
    for bad in (dict(ids=torch.zeros(4, 4, dtype=i32)), dict(w=torch.zeros(4, 3)),
                dict(dst=torch.zeros(4, 8, dtype=i32))):
        with pytest.raises(ValueError):
            route(**bad)
    # (a refused product asked the library first, about no rows)
    assert [a[6] for n, a in calls if n == "nebw_gemm_grouped"] == [4, 4, 0, 0, 0]
    assert len(calls) == 9


def test_route_without_a_workspace(host_calls):
    """A call that needs no workspace takes none."""
    torch = pytest.importorskip("torch")
    import nebw
    d, calls = host_calls
    i32 = torch.int32
    outs = (torch.zeros(4, 2, dtype=i32), torch.zeros(4, 2), torch.zeros(9, dtype=i32),
            torch.zeros(8, dtype=i32), torch.zeros(4, 2, dtype=i32))
    for ws, want in ((None, (None, 0)), (torch.zeros(0), (0, 0))):
        d.moe_route(torch.zeros(4, 8), 4, 8, 2, *outs, ws)
        assert calls[-1][1][-3:-1] == want
    ws = torch.zeros(12, 2)
    d.moe_route(torch.zeros(4, 8), 4, 8, 2, *outs, ws)
    assert calls[-1][1][-3:-1] == (ws.data_ptr(), 96)
    with pytest.raises(TypeError):
        d.moe_route(torch.zeros(4, 8), 4, 8, 2, *outs, ws.t())


@pytest.mark.parametrize("heads,head_dim", [(2, 32), (2, 16), (1, 48), (4, 14)])
def test_heads_of_another_width_are_refused(heads, head_dim):
    """Heads made for one width are not read as so many narrower ones, with the
    first part of a norm's weights."""
    torch = pytest.importorskip("torch")
    import nebw
    side = nebw.Heads.of(torch.zeros(4, 96), heads, gamma=torch.ones(96 // heads))
    side.gpu = 0
    d = nebw.Device.__new__(nebw.Device)
    d.h, d.index = None, 0
    assert d._heads_dtype(side, None, None, 4, 96 // heads) == nebw.F32
    for q, k in ((side, None), (None, side)):
        with pytest.raises(nebw.NebwError, match=f"head_dim {head_dim}") as e:
            d._heads_dtype(q, k, None, 4, head_dim)
        assert e.value.code == 1


def test_operands_of_another_gpu_or_too_few_are_refused():
    """The argument checks of the device calls, on a handle without a device
    and tensors that only say where they are."""
    torch = pytest.importorskip("torch")
    import nebw

    class On:
        dtype = torch.int32

        def __init__(self, gpu, n=4, whole=True):
            self.gpu, self.n, self.whole = gpu, n, whole

        def get_device(self):
            return self.gpu

        def is_contiguous(self):
            return self.whole

        def numel(self):
            return self.n

        def data_ptr(self):
            return 64

    d = nebw.Device.__new__(nebw.Device)
    d.h, d.index = None, 1
    assert d._i32(On(1), 4) == 64 and d._i32(None, 4) is None and d._i32(80, 4) == 80
    for bad in (On(0), On(-1), On(1, whole=False)):
        with pytest.raises(TypeError):
            d._i32(bad)
    with pytest.raises(TypeError):
        d._f32(On(1))
    with pytest.raises(ValueError):
        d._i32(On(1), 5)
    side = nebw.Heads.of(torch.zeros(4, 96), 2)
    with pytest.raises(TypeError):  # host memory
        d._heads_dtype(side, None, None, 4, 48)
    side.gpu = 1
    assert d._heads_dtype(side, None, None, 4, 48) == nebw.F32
    for rows, dim in ((5, 48), (4, 50)):
        with pytest.raises(ValueError):
            d._heads_dtype(None, side, None, rows, dim)
