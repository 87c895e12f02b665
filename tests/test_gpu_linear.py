"""GPU tests of the linear layer against its 64-bit form, with derived bounds (layer_ref.py)."""
from __future__ import annotations

import pytest
import torch

import layer_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(seed, shape, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def _case(dev, rows, k, n, dtype, out_dtype=None, act=0, bias=F32, res=None, seed=0):
    import mbrt

    out_dtype = out_dtype or dtype
    say(f"linear rows={rows} k={k} n={n} {dtype} out={out_dtype} act={act} bias={bias} res={res}")
    x, w = _rand(seed, (rows, k), dtype), _rand(seed + 1, (n, k), dtype, std=1.0 / max(k, 1) ** 0.5)
    b = _rand(seed + 2, (n,), bias, 0.5) if bias else None
    r = _rand(seed + 3, (rows, n), res) if res else None
    got = mbrt.linear(x, w, b, act=act, residual=r, out_dtype=out_dtype)
    torch.cuda.synchronize()
    want, bound = ref.linear(x, w, b, act, r, out_dtype)
    ref.check(got, want, bound, f"linear [{rows}, {k}] -> {n}")


# each form's edges: strips of either operand (up to 64 of the other), 64- and 128-wide tiles, whole and cut
SIZES = [(1, 1, 1), (1, 384, 1536), (5, 7, 3), (16, 64, 16), (17, 65, 33), (60, 384, 1536), (64, 128, 64),
         (65, 64, 65), (65, 63, 66), (64, 1536, 384), (1000, 384, 8), (333, 130, 17), (129, 384, 200), (801, 118, 384),
         (200, 1536, 384), (257, 100, 129), (127, 8, 1), (1, 8, 127), (700, 37, 63)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_sizes(dev, rows, k, n, dtype):
    _case(dev, rows, k, n, dtype, seed=rows + k + n)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k,n", [(2500, 384, 1536), (4133, 200, 1031), (2560, 128, 1664)])
def test_large_tiles(dev, rows, k, n, dtype):
    _case(dev, rows, k, n, dtype, res=dtype, seed=3)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k,n", [(16500, 384, 9), (16400, 96, 5), (6, 385, 16500), (5000, 130, 24), (5001, 66, 40),
                                      (30, 131, 4200), (50, 129, 49200)])
def test_short_operands(dev, rows, k, n, dtype):
    """Many rows against few columns and the other way round: strips and small tiles, in rows at every alignment."""
    _case(dev, rows, k, n, dtype, res=dtype, seed=rows)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k,n", [(700, 840, 390), (700, 328, 390), (650, 256, 448), (1500, 1544, 900), (700, 768, 385)])
def test_few_tiles(dev, rows, k, n, dtype):
    """Tiles whose steps are shared out among groups of waves, whole and cut by the rows' end."""
    _case(dev, rows, k, n, dtype, act=1, res=dtype, seed=n)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("out", [F16, F32])
@pytest.mark.parametrize("rows,k,n", [(33, 67, 41), (700, 129, 131), (2600, 64, 1537), (90, 7, 129)])
def test_odd_rows_in_and_out(dev, rows, k, n, dtype, out):
    _case(dev, rows, k, n, dtype, out, act=2, res=out, seed=9)


@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F32), (F32, F16), (BF16, F32)])
@pytest.mark.parametrize("rows,k,n", [(3, 96, 70), (150, 96, 70), (90, 96, 8)])
def test_epilogue(dev, rows, k, n, dtype, out, act):
    _case(dev, rows, k, n, dtype, out, act=act, bias=BF16, res=BF16, seed=act)
    _case(dev, rows, k, n, dtype, out, act=act, bias=None, res=F32, seed=act + 10)
    _case(dev, rows, k, n, dtype, out, act=act, bias=F16, res=None, seed=act + 20)


def test_activations_far_out(dev):
    """Arguments far into the tails, where the functions saturate."""
    import mbrt

    x = torch.tensor([[-200.0], [-20.0], [-5.0], [-1e-3], [0.0], [1e-3], [5.0], [20.0], [200.0]], device="cuda")
    w = torch.ones((70, 1), device="cuda")
    for act in range(1, 5):
        want, bound = ref.linear(x, w, None, act, None, F32)
        ref.check(mbrt.linear(x, w, act=act), want, bound, f"act {act}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k,n", [(20, 40, 90), (300, 72, 100), (100, 72, 12)])
def test_strides_and_alignment(dev, rows, k, n, dtype):
    """Rows inside wider ones whose other columns hold NaN, odd offsets, and what lies around out untouched."""
    import mbrt

    for pad, off in ((8, 8), (3, 1), (5, 2)):
        say(f"strided linear rows={rows} k={k} n={n} pad={pad} off={off}")
        big = torch.full((rows, k + pad), float("nan"), dtype=dtype, device="cuda")
        at = min(off, pad)
        x = big[:, at:at + k]
        x.copy_(_rand(1, (rows, k), dtype))
        wbig = torch.full((n, k + pad), float("nan"), dtype=dtype, device="cuda")
        w = wbig[:, at:at + k]
        w.copy_(_rand(2, (n, k), dtype, 0.2))
        rbig = torch.full((rows, n + pad), float("nan"), dtype=dtype, device="cuda")
        r = rbig[:, at:at + n]
        r.copy_(_rand(3, (rows, n), dtype))
        obig = torch.full((rows + 1, n + pad), 7.0, dtype=dtype, device="cuda")
        out = obig[:rows, at:at + n]
        mbrt.linear(x, w, None, out, residual=r)
        want, bound = ref.linear(x, w, None, 0, r, dtype)
        ref.check(out, want, bound, "strided")
        assert bool((obig[rows] == 7).all() and (obig[:, :at] == 7).all() and (obig[:, at + n:] == 7).all())


def test_leading_dims_broadcast_rows_and_in_place(dev):
    import mbrt

    x = _rand(1, (3, 50, 64), BF16)
    w, b = _rand(2, (80, 64), BF16, 0.1), _rand(3, (80,), F32)
    stream_ = _rand(4, (3, 50, 80), BF16)
    want, bound = ref.linear(x.view(150, 64), w, b, 0, stream_.view(150, 80).clone(), BF16)
    got = mbrt.linear(x, w, b, stream_, residual=stream_)   # the residual stream updated in place
    assert got is stream_
    ref.check(stream_.view(150, 80), want, bound, "in place")
    one = _rand(5, (1, 64), BF16).expand(130, 64)            # one row, 130 times
    want, bound = ref.linear(one, w, None, 0, None, BF16)
    ref.check(mbrt.linear(one, w), want, bound, "broadcast rows")


def test_empty_and_zero_sizes(dev):
    import mbrt

    w, b = _rand(1, (5, 8), F32), _rand(2, (5,), F32)
    assert mbrt.linear(torch.empty((0, 8), device="cuda"), w, b).shape == (0, 5)
    assert mbrt.linear(torch.empty((4, 8), device="cuda"), w[:0]).shape == (4, 0)
    got = mbrt.linear(torch.empty((70, 0), device="cuda"), torch.empty((5, 0), device="cuda"), b, act=3)
    want = torch.sigmoid(b.cpu().double()).expand(70, 5)
    ref.check(got, want, 16 * ref.U + 0 * want, "no features")


@pytest.mark.parametrize("rows,n", [(7, 90), (200, 90), (200, 5)])
def test_specials_stay_in_their_row_and_column(dev, rows, n):
    import mbrt

    x, w = _rand(1, (rows, 80), BF16), _rand(2, (n, 80), BF16)
    x[3, 79] = float("nan")
    w[4, 0] = float("inf")
    got = mbrt.linear(x, w).cpu()
    bad = torch.zeros((rows, n), dtype=torch.bool)
    bad[3] = True
    bad[:, 4] = True
    assert bool((~torch.isfinite(got) == bad).all())


def test_rows_far_apart(dev):
    """Offsets beyond 32 bits, in bytes and in elements."""
    import mbrt

    rows, k, n, stride = 70000, 24, 8, 32768
    big = torch.empty(rows * stride, dtype=BF16, device="cuda")
    x = big.as_strided((rows, k), (stride, 1))
    x.copy_(_rand(1, (rows, k), BF16))
    w = _rand(2, (n, k), BF16)
    w2 = _rand(3, (80, k), BF16)
    for weight in (w, w2):
        got = mbrt.linear(x, weight)
        want, bound = ref.linear(x.contiguous(), weight, None, 0, None, BF16)
        ref.check(got, want, bound, "far rows")


def test_same_result_every_time_captured_and_on_another_stream(dev):
    import mbrt

    x, w, b = _rand(1, (300, 384), BF16), _rand(2, (390, 384), BF16, 0.05), _rand(3, (390,), F32)
    xs = _rand(4, (9, 384), BF16)
    want, small = mbrt.linear(x, w, b, act=2), mbrt.linear(xs, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = mbrt.linear(x, w, b, act=2, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    out, outs = torch.empty_like(want), torch.empty_like(small)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mbrt.linear(x, w, b, out, act=2)
        mbrt.linear(xs, w, b, outs)
    for i in range(4):
        out.zero_(), outs.zero_()
        graph.replay()
        eager = mbrt.linear(x, w, b, act=2)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(outs, small) and torch.equal(eager, want), i


def _arguments(dtype):
    big = 6e4 if dtype == F16 else 1e30
    inf = float("inf")
    return torch.tensor([-inf, -big, -200.0, -12.0, -6.5, -5.0, -3.75, -1.0, -0.125, -1e-3, 0.0, 1e-3, 0.3125, 2.5, 6.0, 20.0,
                         1000.0, big, inf, float("nan")], dtype=dtype)


# one argument per row of x, in column 0, whose weights are 1: strips and tiles, whole pieces and cut ones, no features
@pytest.mark.parametrize("rows,k,n", [(20, 64, 70), (20, 7, 70), (1500, 72, 200), (1500, 65, 200), (9, 0, 20)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
def test_activations_of_infinities_and_nan(dev, rows, k, n, dtype, out, act):
    """Arguments that are infinite or NaN give what the functions' formulas give, for every type of operand and result."""
    import mbrt

    say(f"special arguments rows={rows} k={k} n={n} {dtype} -> {out} act={act}")
    v = _arguments(dtype)
    if k == 0:
        x, w, b = torch.empty((rows, 0), dtype=dtype, device="cuda"), torch.empty((n, 0), dtype=dtype, device="cuda"), v.cuda()
        arg = v.expand(rows, n)
    else:
        x, w, b = torch.zeros((rows, k), dtype=dtype), torch.zeros((n, k), dtype=dtype, device="cuda"), None
        x[:, 0] = v.repeat(rows // v.numel() + 1)[:rows]
        w[:, 0] = 1
        arg, x = x[:, :1].expand(rows, n), x.cuda()
    got = mbrt.linear(x, w, b, act=act, out_dtype=out).cpu().double()
    want, _ = ref.activation(arg, act, out, False)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    special = torch.isinf(arg.double()) & ~torch.isnan(want)
    assert torch.equal(got[special], want[special])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("act", [1, 2, 3, 4])
def test_activations_in_their_tails(dev, dtype, out, act):
    """Values relative to themselves, into the tails: the short forms are for 2-byte results of 2-byte operands alone."""
    import mbrt

    x = torch.cat((torch.linspace(-13, 13, 1301), torch.tensor([-6e4, -200.0, -30.0, 30.0, 200.0, 6e4])))[:, None].to(dtype)
    for n in (5, 200):   # strips and tiles
        say(f"tails {dtype} -> {out} act={act} n={n}")
        w = torch.ones((n, 1), dtype=dtype, device="cuda")
        want, bound = ref.activation(x.expand(-1, n), act, out, dtype != F32 and out != F32)
        ref.check(mbrt.linear(x.cuda(), w, act=act, out_dtype=out), want, bound, f"act {act}")


def test_outputs_beside_their_inputs_and_within_them(dev):
    """Columns of one wider matrix as input and out, and a residual beside out; what shares memory otherwise is refused."""
    import mbrt

    for rows, k, n in ((9, 64, 72), (700, 64, 72), (700, 72, 72)):
        say(f"beside rows={rows} k={k} n={n}")
        wide = _rand(1, (rows, k + 2 * n), BF16)
        x, out, r = wide[:, :k], wide[:, k:k + n], wide[:, k + n:]
        w = _rand(2, (n, k), BF16, 0.1)
        want, bound = ref.linear(x, w, None, 0, r, BF16)
        kept = wide.clone()
        ref.check(mbrt.linear(x, w, out=out, residual=r), want, bound, "beside")
        assert torch.equal(x, kept[:, :k]) and torch.equal(r, kept[:, k + n:])
        with pytest.raises(mbrt.MbrtError, match="overlaps"):
            mbrt.linear(x, w, out=wide[:, k - 1:k - 1 + n])
        if rows == 700:
            with pytest.raises(mbrt.MbrtError, match="overlaps"):
                mbrt.linear(r, _rand(2, (n, n), BF16), out=r)
    sq = _rand(3, (64, 64), BF16)
    for kw in (dict(out=sq), dict(residual=sq[:1].expand(64, 64), out=sq)):
        with pytest.raises(mbrt.MbrtError, match="overlaps"):
            mbrt.linear(sq if len(kw) == 1 else _rand(4, (64, 64), BF16), _rand(5, (64, 64), BF16), **kw)
    with pytest.raises(mbrt.MbrtError, match="overlaps"):
        mbrt.linear(_rand(4, (64, 64), BF16), sq, out=sq)


def test_calls_without_the_extension_module(dev, monkeypatch):
    """The same results, and the same refusals on the GPU, through ctypes."""
    import mbrt
    from mbrt import _calls

    wide = _rand(1, (3, 40, 100), BF16)
    x, w, b, r = wide[..., :64], _rand(2, (36, 64), BF16, 0.1), _rand(3, (36,), F32), _rand(4, (3, 40, 36), F16)
    want = mbrt.linear(x, w, b, wide[..., 64:].clone(), act=2, residual=r)
    monkeypatch.setattr(mbrt, "_n", _calls)
    assert torch.equal(mbrt.linear(x, w, b, wide[..., 64:], act=2, residual=r), want)
    with pytest.raises(mbrt.MbrtError, match="overlaps"):
        mbrt.linear(x, w, b, wide[..., 63:99])
