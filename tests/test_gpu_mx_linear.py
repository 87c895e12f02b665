"""GPU tests of the 4-bit linear layer against its 64-bit form, with derived bounds (mx_ref.py)."""
from __future__ import annotations

import math

import pytest
import torch

import layer_ref
import mx_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
MX = "mx"


def _rand(seed, shape, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def _operand(seed, shape, kind, std=1.0):
    """x of a kind, and its values in 64 bits."""
    import mbrt

    if kind == MX:
        # blocks of very different sizes
        x = _rand(seed, shape, F32, std) * torch.exp2(4 * _rand(seed + 50, (*shape[:-1], 1), F32)).round()
        held = mbrt.mx_quantize(x)
        return held, ref.held(held)
    x = _rand(seed, shape, kind, std)
    return x, x.cpu().double()


def _check(got, x64, w64, b, act, r, out, what):
    torch.cuda.synchronize()
    want, bound = ref.linear(x64, w64, b, act, r, None if out == MX else out)
    if out == MX:
        ref.check_held(got, want, bound, what)
    else:
        layer_ref.check(got, want, bound, what)


def _case(dev, rows, k, n, x, out=None, act=0, bias=F32, res=None, seed=0):
    import mbrt

    out = out or (BF16 if x == MX else x)
    say(f"mx_linear rows={rows} k={k} n={n} x={x} out={out} act={act} bias={bias} res={res}")
    xs, x64 = _operand(seed, (rows, k), x)
    w, w64 = _operand(seed + 1, (n, k), MX, 1.0 / max(k, 1) ** 0.5)
    b = _rand(seed + 2, (n,), bias, 0.5) if bias else None
    r = _rand(seed + 3, (rows, n), res) if res else None
    got = mbrt.mx_linear(xs, w, b, act=act, residual=r, out_dtype=mbrt.MxTensor if out == MX else out)
    _check(got, x64, w64, b, act, r, out, f"mx_linear [{rows}, {k}] -> {n}")


SIZES = [(1, 1, 1), (1, 384, 1536), (5, 7, 3), (16, 64, 16), (17, 65, 33), (60, 384, 1536), (64, 128, 64), (65, 64, 65),
         (65, 63, 66), (64, 1536, 384), (1000, 384, 8), (333, 130, 17), (129, 384, 200), (801, 118, 384), (200, 1536, 384),
         (257, 100, 129), (127, 8, 1), (1, 8, 127), (700, 37, 63), (3, 5000, 40), (400, 2081, 700), (1, 8192, 100),
         (33, 513, 64), (2, 96, 4000)]


@pytest.mark.parametrize("x", [MX, BF16, F16, F32])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_sizes(dev, rows, k, n, x):
    _case(dev, rows, k, n, x, seed=rows + k + n)


@pytest.mark.parametrize("x", [MX, BF16, F16, F32])
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (60, 384, 1536), (5, 70, 33), (333, 130, 97), (1000, 100, 8), (400, 384, 700)])
def test_results_in_4_bits(dev, rows, k, n, x):
    _case(dev, rows, k, n, x, MX, act=2, seed=rows)
    _case(dev, rows, k, n, x, MX, act=0, bias=None, res=F16, seed=rows + 9)


@pytest.mark.parametrize("x,out", [(MX, BF16), (MX, MX), (MX, F32), (BF16, BF16), (F16, MX), (F32, F32)])
@pytest.mark.parametrize("rows,k,n", [(2500, 384, 1536), (4133, 200, 1031), (2560, 1100, 1664)])
def test_large_tiles(dev, rows, k, n, x, out):
    _case(dev, rows, k, n, x, out, res=None if out == MX else out, seed=3)


@pytest.mark.parametrize("x", [MX, F16, BF16])
@pytest.mark.parametrize("rows,k,n", [(16500, 384, 9), (16400, 96, 5), (6, 385, 16500), (5000, 130, 24), (5001, 66, 40),
                                      (30, 131, 4200), (50, 129, 20000)])
def test_short_operands(dev, rows, k, n, x):
    _case(dev, rows, k, n, x, res=BF16, seed=rows)


@pytest.mark.parametrize("x", [MX, F16, BF16, F32])
@pytest.mark.parametrize("rows,k,n", [(1, 100, 16400), (2, 545, 16390), (4, 1290, 16411), (16, 513, 8200), (1, 9, 40001)])
def test_few_rows_against_many_weights(dev, rows, k, n, x):
    _case(dev, rows, k, n, x, bias=F16, res=F32, seed=n)
    _case(dev, rows, k, n, x, MX, act=1, seed=n + 9)


@pytest.mark.parametrize("out,res", [(BF16, BF16), (F32, None)])
@pytest.mark.parametrize("rows,k,n", [(4090, 1540, 4001), (3900, 1633, 4096)])
def test_long_k(dev, rows, k, n, out, res):
    _case(dev, rows, k, n, MX, out, act=2 if res else 0, res=res, seed=k)


@pytest.mark.parametrize("x", [F16, BF16, F32])
@pytest.mark.parametrize("rows,k,n", [(520, 63, 640), (520, 64, 640), (500, 129, 650), (513, 384, 900), (400, 1152, 1100), (700, 1007, 530)])
def test_steps_shared_by_groups_of_waves(dev, rows, k, n, x):
    _case(dev, rows, k, n, x, act=2, res=F16, seed=k)


@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("x,out", [(MX, BF16), (MX, F32), (F32, F32), (BF16, F16), (F16, F32)])
@pytest.mark.parametrize("rows,k,n", [(3, 96, 70), (150, 96, 70), (90, 96, 8)])
def test_epilogue(dev, rows, k, n, x, out, act):
    _case(dev, rows, k, n, x, out, act=act, bias=BF16, res=BF16, seed=act)
    _case(dev, rows, k, n, x, out, act=act, bias=None, res=F32, seed=act + 10)
    _case(dev, rows, k, n, x, out, act=act, bias=F16, res=None, seed=act + 20)


@pytest.mark.parametrize("x", [MX, BF16, F16, F32])
@pytest.mark.parametrize("rows,k,n", [(20, 40, 90), (300, 72, 100), (100, 72, 12), (200, 300, 260)])
def test_strides_and_alignment(dev, rows, k, n, x):
    """Rows inside wider ones whose rest is NaN (in codes: anything), and what lies around out untouched."""
    import mbrt

    kb = -(-k // 32)
    for pad, off in ((8, 8), (3, 1), (5, 2)):
        say(f"strided mx_linear rows={rows} k={k} n={n} x={x} pad={pad} off={off}")

        def held_in(count, seed):
            codes = torch.full((count, 16 * kb + 48), 0x77, dtype=torch.uint8, device="cuda")
            scales = torch.full((count, kb + pad), 255, dtype=torch.uint8, device="cuda")
            h = mbrt.MxTensor(codes[:, 16:16 + 16 * kb], scales[:, off % pad:off % pad + kb], k)
            mbrt.mx_quantize(_rand(seed, (count, k), F32, 0.2), out=h)
            return h, ref.held(h)

        w, w64 = held_in(n, 2)
        if x == MX:
            xs, x64 = held_in(rows, 1)
        else:
            big = torch.full((rows, k + pad), math.nan, dtype=x, device="cuda")
            xs = big[:, min(off, pad):min(off, pad) + k]
            xs.copy_(_rand(1, (rows, k), x))
            x64 = xs.cpu().double()
        odt = BF16 if x == MX else x
        rbig = torch.full((rows, n + pad), math.nan, dtype=odt, device="cuda")
        r = rbig[:, min(off, pad):min(off, pad) + n]
        r.copy_(_rand(3, (rows, n), odt))
        obig = torch.full((rows + 1, n + pad), 7.0, dtype=odt, device="cuda")
        at = min(off, pad)
        out = obig[:rows, at:at + n]
        mbrt.mx_linear(xs, w, None, out, residual=r)
        _check(out, x64, w64, None, 0, r, odt, "strided")
        assert bool((obig[rows] == 7).all() and (obig[:, :at] == 7).all() and (obig[:, at + n:] == 7).all())
        nb = -(-n // 32)
        codes = torch.full((rows + 1, 16 * nb + 32), 0x5A, dtype=torch.uint8, device="cuda")
        scales = torch.full((rows + 1, nb + 3), 0x5A, dtype=torch.uint8, device="cuda")
        held = mbrt.MxTensor(codes[:rows, 16:16 + 16 * nb], scales[:rows, 1:1 + nb], n)
        mbrt.mx_linear(xs, w, None, held, residual=r)
        _check(held, x64, w64, None, 0, r, MX, "strided")
        assert bool((codes[:, :16] == 0x5A).all() and (codes[:, 16 + 16 * nb:] == 0x5A).all() and (codes[rows] == 0x5A).all())
        assert bool((scales[:, :1] == 0x5A).all() and (scales[:, 1 + nb:] == 0x5A).all() and (scales[rows] == 0x5A).all())


def test_leading_dims_broadcast_rows_and_in_place(dev):
    import mbrt

    x, x64 = _operand(1, (3, 50, 64), MX)
    w, w64 = _operand(2, (80, 64), MX, 0.1)
    b = _rand(3, (80,), F32)
    stream_ = _rand(4, (3, 50, 80), BF16)
    want, bound = ref.linear(x64.view(150, 64), w64, b, 0, stream_.view(150, 80).clone(), BF16)
    assert mbrt.mx_linear(x, w, b, stream_, residual=stream_) is stream_
    layer_ref.check(stream_.view(150, 80), want, bound, "in place")
    one = _rand(5, (1, 64), BF16).expand(130, 64)
    want, bound = ref.linear(one, w64, None, 0, None, BF16)
    layer_ref.check(mbrt.mx_linear(one, w), want, bound, "broadcast rows")


def test_empty_and_zero_sizes(dev):
    import mbrt

    w, _ = _operand(1, (5, 8), MX)
    b = _rand(2, (5,), F32)
    assert mbrt.mx_linear(torch.empty((0, 8), device="cuda"), w, b).shape == (0, 5)
    none = mbrt.MxTensor(w.codes[:0], w.scales[:0], 8)
    assert mbrt.mx_linear(torch.empty((4, 8), device="cuda"), none).shape == (4, 0)
    w0 = mbrt.mx_empty((5, 0))
    want = torch.sigmoid(b.cpu().double()).expand(70, 5)
    for x in (torch.empty((70, 0), device="cuda"), mbrt.mx_empty((70, 0))):
        got = mbrt.mx_linear(x, w0, b, act=3, out_dtype=F32)
        layer_ref.check(got, want, 16 * ref.U + 0 * want, "no features")
        ref.check_held(mbrt.mx_linear(x, w0, b, act=3, out_dtype=mbrt.MxTensor), want, 16 * ref.U + 0 * want, "no features")
    w1 = mbrt.mx_empty((1101, 0))
    b1 = _rand(3, (1101,), F32)
    want = b1.cpu().double().expand(3, 1101)
    ref.check_held(mbrt.mx_linear(mbrt.mx_empty((3, 0)), w1, b1, out_dtype=mbrt.MxTensor), want, 0 * want, "no features, wide")


@pytest.mark.parametrize("x", [MX, BF16, F16, F32])
@pytest.mark.parametrize("rows,n", [(7, 90), (200, 90), (200, 5), (600, 300)])
def test_specials_stay_in_their_row_and_column(dev, rows, n, x):
    import mbrt

    v, w = _rand(1, (rows, 80), F32), _rand(2, (n, 80), F32)
    v[3, 79], w[4, 0] = math.nan, math.inf
    xs = mbrt.mx_quantize(v) if x == MX else v.to(x)
    got = mbrt.mx_linear(xs, mbrt.mx_quantize(w), out_dtype=F32).cpu()
    bad = torch.zeros((rows, n), dtype=torch.bool)
    bad[3], bad[:, 4] = True, True
    assert torch.equal(torch.isnan(got), bad)


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("x", [MX, BF16, F16, F32])
@pytest.mark.parametrize("rows,n", [(7, 90), (200, 160), (600, 400), (5000, 1024)])
def test_specials_in_4_bits(dev, rows, n, x, act):
    """A NaN takes its block along, its scale 255, and no other; so does an infinity that act leaves one, or makes NaN."""
    import mbrt

    v, w = _rand(1, (rows, 80), F32), _rand(2, (n, 80), F32, 0.1)
    b = _rand(3, (n,), F32)
    v[3, 7], b[33], b[70] = math.nan, math.inf, -math.inf
    xs = mbrt.mx_quantize(v) if x == MX else v.to(x)
    w = mbrt.mx_quantize(w)
    got = mbrt.mx_linear(xs, w, b, act=act, out_dtype=mbrt.MxTensor).scales.cpu()
    bad = torch.zeros((rows, -(-n // 32)), dtype=torch.bool)
    bad[3] = True
    if act < 3:
        bad[:, 1] = bad[:, 2] = True
    assert torch.equal(got == 255, bad)


@pytest.mark.parametrize("x", [BF16, F16, F32])
@pytest.mark.parametrize("rows,n", [(3, 40), (300, 200)])
def test_infinities_of_x(dev, rows, n, x):
    """An infinity meets a weight that is not zero: it stays one, in its sign."""
    import mbrt

    v = torch.zeros((rows, 40), dtype=x, device="cuda")
    v[0, 0], v[1, 0], v[2, 39] = math.inf, -math.inf, math.inf
    w = torch.ones((n, 40), device="cuda")
    w[:, 39] = -2
    got = mbrt.mx_linear(v, mbrt.mx_quantize(w), out_dtype=F32).cpu()
    assert bool((got[0] == math.inf).all() and (got[1] == -math.inf).all() and (got[2] == -math.inf).all() and (got[3:] == 0).all())


@pytest.mark.parametrize("rows,n", [(2, 40), (300, 200)])
def test_f32_products_are_exact(dev, rows, n):
    """One weight that is not zero per row: its product with all 24 bits of x, over most exponents."""
    import mbrt

    g = torch.Generator().manual_seed(1)
    x = torch.randn((rows, 70), generator=g) * torch.exp2(torch.randint(-60, 60, (rows, 70), generator=g).float())
    w = torch.zeros((n, 70))
    w[torch.arange(n), torch.arange(n) % 70] = 1.5
    got = mbrt.mx_linear(x.cuda(), mbrt.mx_quantize(w.cuda())).cpu()
    want = x.double()[:, torch.arange(n) % 70] * 1.5
    assert bool(((got.double() - want).abs() <= 2.0 ** -23 * want.abs()).all())


@pytest.mark.parametrize("x", [MX, BF16])
def test_scales_at_their_ends(dev, x):
    """The smallest and largest scales on one side against ordinary ones on the other."""
    import mbrt

    for e in (-110, -60, 60, 110):
        say(f"scales around 2^{e} x={x}")
        xs, x64 = _operand(1, (40, 96), x)
        w = mbrt.mx_quantize(_rand(2, (50, 96), F32) * 2.0 ** e)
        want, bound = ref.linear(x64, ref.held(w), None, 0, None, F32)
        layer_ref.check(mbrt.mx_linear(xs, w, out_dtype=F32), want, bound, f"2^{e}")


def test_rows_far_apart(dev):
    """Offsets beyond 32 bits, in bytes and in elements; strides that tiles do not take."""
    import mbrt

    rows, k, stride = 70000, 64, 65536
    big = torch.empty(rows * stride, dtype=torch.uint8, device="cuda")
    held = mbrt.MxTensor(big.as_strided((rows, 32), (stride, 1)), big[64:].as_strided((rows, 2), (stride, 1)), k)
    mbrt.mx_quantize(_rand(1, (rows, k), BF16), out=held)
    x64 = ref.held(held)
    for n in (8, 80, 200):
        w, w64 = _operand(2, (n, k), MX)
        want, bound = ref.linear(x64, w64, None, 0, None, BF16)
        layer_ref.check(mbrt.mx_linear(held, w), want, bound, "far rows")
    apart = 1 << 22
    few = mbrt.MxTensor(big.as_strided((900, 32), (apart, 1)), big[64:].as_strided((900, 2), (apart, 1)), k)
    mbrt.mx_quantize(_rand(1, (900, k), BF16), out=few)
    w, w64 = _operand(2, (400, k), MX)
    want, bound = ref.linear(ref.held(few), w64, None, 0, None, BF16)
    layer_ref.check(mbrt.mx_linear(few, w), want, bound, "rows 4 MB apart")


def test_same_result_every_time_captured_and_on_another_stream(dev):
    import mbrt

    x, _ = _operand(1, (300, 384), MX)
    xs, xb = _operand(4, (9, 384), MX)[0], _rand(5, (9, 384), BF16)
    w, _ = _operand(2, (390, 384), MX, 0.05)
    b = _rand(3, (390,), F32)
    calls = [lambda o, s=None: mbrt.mx_linear(x, w, b, o, act=2, stream=s), lambda o, s=None: mbrt.mx_linear(xs, w, b, o, stream=s),
             lambda o, s=None: mbrt.mx_linear(xb, w, b, o, stream=s)]
    want = [c(None) for c in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [c(None, side) for c in calls]
    side.synchronize()
    assert all(torch.equal(g, t) for g, t in zip(got, want))
    outs = [torch.empty_like(t) for t in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c, o in zip(calls, outs):
            c(o)
    for i in range(4):
        for o in outs:
            o.zero_()
        graph.replay()
        eager = [c(None) for c in calls]
        torch.cuda.synchronize()
        assert all(torch.equal(o, t) and torch.equal(e, t) for o, e, t in zip(outs, eager, want)), i


def test_outputs_within_their_inputs_are_refused(dev):
    import mbrt

    x, _ = _operand(1, (70, 64), MX)
    w, _ = _operand(2, (64, 64), MX)
    wide = _rand(3, (70, 136), BF16)
    for kw in (dict(out=x), dict(out=mbrt.MxTensor(w.codes, x.scales[:64], 64))):
        with pytest.raises(mbrt.MbrtError, match="overlaps"):
            mbrt.mx_linear(x if kw["out"] is x else mbrt.MxTensor(x.codes[:64], x.scales[:64], 64), w, **kw)
    with pytest.raises(mbrt.MbrtError, match="overlaps"):
        mbrt.mx_linear(wide[:, :64], w, out=wide[:, 63:127])
    kept = wide.clone()
    want = mbrt.mx_linear(wide[:, :64].contiguous(), w)
    mbrt.mx_linear(wide[:, :64], w, out=wide[:, 64:128])
    assert torch.equal(wide[:, 64:128], want) and torch.equal(wide[:, :64], kept[:, :64]) and torch.equal(wide[:, 128:], kept[:, 128:])


def test_calls_without_the_extension_module(dev, monkeypatch):
    import mbrt
    from mbrt import _calls

    x, _ = _operand(1, (3, 40, 100), MX)
    xb = _rand(7, (3, 40, 100), F16)
    w, _ = _operand(2, (36, 100), MX, 0.1)
    b, r = _rand(3, (36,), F32), _rand(4, (3, 40, 36), F16)
    run = lambda: [mbrt.mx_linear(x, w, b, act=2, residual=r), mbrt.mx_linear(xb, w, b, residual=r),
                   *mbrt.mx_linear(x, w, b, out_dtype=mbrt.MxTensor)[:2]]
    want = run()
    monkeypatch.setattr(mbrt, "_n", _calls)
    assert all(torch.equal(g, t) for g, t in zip(run(), want))
