"""GPU tests of the 4-bit quantisation and its inverse, bit for bit against their 64-bit forms (mx_ref.py)."""
from __future__ import annotations

import math

import pytest
import torch

import mx_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def _rand(seed, shape, dtype):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * torch.exp(2 * torch.randn((*shape[:-1], 1), generator=g))).to(dtype).cuda()


def _check(got, x, what=""):
    codes, scales = ref.quantize(x)
    assert torch.equal(got.scales.cpu().long(), scales), what
    fine = (scales != 255)[..., None].expand(*scales.shape, 32).flatten(-2)
    assert torch.equal(ref.unpack(got.codes)[fine], codes[fine]), what


def _back(held, x, dtype):
    import mbrt

    got = mbrt.mx_dequantize(held, out_dtype=dtype)
    want = ref.held(held).to(dtype)
    assert torch.equal(got.cpu().nan_to_num(7e4), want.nan_to_num(7e4))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 32), (3, 31), (5, 33), (17, 64), (801, 118), (60, 384), (7, 1001), (2, 4096),
                                    (3000, 40), (129, 1536), (1, 100003)])
def test_sizes(dev, rows, n, dtype):
    import mbrt

    say(f"mx_quantize [{rows}, {n}] {dtype}")
    x = _rand(rows + n, (rows, n), dtype)
    held = mbrt.mx_quantize(x)
    assert held.shape == (rows, n) and held.codes.shape == (rows, 16 * math.ceil(n / 32))
    _check(held, x)
    for out in TYPES:
        _back(held, x, out)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_value(dev, dtype):
    """Every 2-byte value, alone in its block and beside a larger one: subnormals, infinities and NaN too."""
    import mbrt

    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    for beside in (0.0, 1.0, 6e4):
        say(f"every {dtype} beside {beside}")
        x = torch.zeros((65536, 32), dtype=dtype)
        x[:, 5], x[:, 30] = v, beside
        x = x.cuda()
        _check(mbrt.mx_quantize(x), x)


def test_borders_in_f32(dev):
    """Values at, below and above each border, over the whole range of exponents."""
    import mbrt

    border = torch.tensor([0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0, 7.999])
    rows = []
    for e in [-149, -140, -130, -128, -127, -126, -125, -124, -100, -2, -1, 0, 1, 50, 100, 124, 125]:
        b = torch.ldexp(border.double(), torch.tensor(e)).float()
        for t in (b, torch.nextafter(b, torch.tensor(0.0)), torch.nextafter(b, torch.tensor(math.inf))):
            rows.append(torch.cat((t, -t)))
    x = torch.stack(rows).cuda()
    _check(mbrt.mx_quantize(x), x)
    _back(mbrt.mx_quantize(x), x, F32)


def test_every_code_under_every_scale(dev):
    import mbrt

    codes = torch.arange(256).repeat(256, 1).to(torch.uint8).cuda()           # 16 blocks of every byte
    scales = torch.arange(256)[:, None].expand(256, 16).to(torch.uint8).contiguous().cuda()
    held = mbrt.MxTensor(codes, scales, 512)
    for dtype in TYPES:
        _back(held, None, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan(dev, dtype):
    import mbrt

    x = _rand(1, (8, 100), dtype)
    x[1, 3], x[2, 40], x[3, 99], x[4, 64:96] = math.nan, math.inf, -math.inf, 0
    held = mbrt.mx_quantize(x)
    _check(held, x)
    y = mbrt.mx_dequantize(held).cpu()
    bad = torch.zeros((8, 100), dtype=torch.bool)
    bad[1, :32], bad[2, 32:64], bad[3, 96:] = True, True, True
    assert torch.equal(torch.isnan(y), bad) and bool((y[4, 64:96] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,pad,off", [(64, 8, 8), (64, 3, 1), (45, 5, 2), (33, 1, 0)])
def test_strides_and_what_lies_around(dev, dtype, n, pad, off):
    import mbrt

    rows, blocks = 50, -(-n // 32)
    say(f"strided mx n={n} pad={pad} off={off} {dtype}")
    big = torch.full((rows, n + pad), math.nan, dtype=dtype, device="cuda")
    x = big[:, off:off + n]
    x.copy_(_rand(2, (rows, n), dtype))
    codes = torch.full((rows + 1, 16 * blocks + 32), 0x5A, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows + 1, blocks + 3), 0x5A, dtype=torch.uint8, device="cuda")
    held = mbrt.MxTensor(codes[:rows, 16:16 + 16 * blocks], scales[:rows, 1:1 + blocks], n)
    assert mbrt.mx_quantize(x, out=held) is held
    _check(held, x)
    assert bool((codes[:, :16] == 0x5A).all() and (codes[:, 16 + 16 * blocks:] == 0x5A).all() and (codes[rows] == 0x5A).all())
    assert bool((scales[:, :1] == 0x5A).all() and (scales[:, 1 + blocks:] == 0x5A).all() and (scales[rows] == 0x5A).all())
    out = torch.full((rows + 1, n + pad), 7.0, dtype=dtype, device="cuda")
    mbrt.mx_dequantize(held, out[:rows, off:off + n])
    assert torch.equal(out[:rows, off:off + n].cpu(), ref.held(held).to(dtype))
    assert bool((out[rows] == 7).all() and (out[:, :off] == 7).all() and (out[:, off + n:] == 7).all())


def test_leading_dims_empty_and_broadcast(dev):
    import mbrt

    x = _rand(1, (3, 5, 70), BF16)
    held = mbrt.mx_quantize(x)
    assert held.shape == (3, 5, 70)
    _check(held, x)
    assert mbrt.mx_dequantize(held).shape == (3, 5, 70)
    assert mbrt.mx_quantize(x[:0]).codes.shape == (0, 5, 48)
    assert mbrt.mx_quantize(x[..., :0]).codes.shape == (3, 5, 0)
    one = x[0, :1].expand(9, 70)
    _check(mbrt.mx_quantize(one), one)


def test_rows_far_apart(dev):
    """Offsets beyond 32 bits, in bytes and in elements, on both sides."""
    import mbrt

    rows, n, stride = 70000, 40, 65536
    big = torch.empty(rows * stride, dtype=BF16, device="cuda")
    x = big.as_strided((rows, n), (stride, 1))
    x.copy_(_rand(1, (rows, n), BF16))
    held = mbrt.mx_quantize(x)
    _check(held, x)
    want = mbrt.mx_dequantize(held)
    x.zero_()
    mbrt.mx_dequantize(held, x)
    assert torch.equal(x, want)


def test_captured_and_on_another_stream(dev):
    import mbrt

    x = _rand(1, (300, 384), BF16)
    want = mbrt.mx_quantize(x)
    back = mbrt.mx_dequantize(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = mbrt.mx_quantize(x, stream=side)
    gback = mbrt.mx_dequantize(got, stream=side)
    side.synchronize()
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales) and torch.equal(gback, back)
    held, out = mbrt.mx_empty((300, 384)), torch.empty_like(back)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mbrt.mx_quantize(x, out=held)
        mbrt.mx_dequantize(held, out)
    for i in range(3):
        x.copy_(_rand(10 + i, (300, 384), BF16))
        out.zero_()
        graph.replay()
        eager = mbrt.mx_dequantize(mbrt.mx_quantize(x))
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i


def test_native_and_ctypes_calls_agree(dev, monkeypatch):
    import mbrt
    from mbrt import _calls

    x = _rand(4, (3, 40, 77), F16)
    want = mbrt.mx_quantize(x)
    back = mbrt.mx_dequantize(want, out_dtype=F32)
    monkeypatch.setattr(mbrt, "_n", _calls)
    got = mbrt.mx_quantize(x)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    assert torch.equal(mbrt.mx_dequantize(got, out_dtype=F32), back)
