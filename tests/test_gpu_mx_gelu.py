"""GPU tests of GELU in front of results in 4 bits: its values in the negative tail, where a block's codes go by how
exact each value is relative to itself."""
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


def _gelu(pre, act):
    """(value, bound) of x Phi(s x), s sqrt 2 (act 1) or 1 (act 2), evaluated in f32 by exp2 of -k x^2 and a scaled tail.

    Roundings, in halves of U = 2^-23: k, its product with |x| and that with |x| each move the exponent, (s x)^2 / 2 as a natural
    one, by one of its size: 0.75 (s x)^2 U.  The argument 1 + c |x| (1), its reciprocal (2, and as much again in the polynomial),
    the polynomial of degree 7 with a sum of magnitudes of at most twice its value (7 steps: 14 at most), what it differs from the
    function by (2.3e-8 of 0.12 and more: 4), exp2 (2), three products and the last sum (4): 29 halves, taken as 32.  What lies below
    f32's normal numbers may be 0."""
    y, _ = layer_ref.act64(pre, act)
    z2 = (2.0 if act == 1 else 1.0) * pre * pre
    tail = 0.5 * pre.abs() * torch.special.erfc(torch.sqrt(z2 / 2))
    return y, ref.U * ((0.75 * z2 + 16) * tail + 0.5 * y.abs()) + pre.abs() * 2.0 ** -126


def _run(rows, n, x, act, mean, std):
    """act(x I + bias): x and bias on a grid of 2^-10, so that every sum is exact and what differs is the function."""
    import mbrt

    say(f"mx_linear GELU {act} around {mean} rows={rows} n={n} x={x}")
    s = math.sqrt(0.5) if act == 1 else 1.0
    k = 64                       # column j has the feature j % k
    g = torch.Generator().manual_seed(rows + act)
    v = torch.randn((rows, k), generator=g) * (0.6 * std * s)
    if x == MX:
        xs = mbrt.mx_quantize(v.cuda())
        x64 = ref.held(xs)
    else:
        xs = (torch.round(v * 64) / 64).clamp(-3.875, 3.875).to(x).cuda()
        x64 = xs.cpu().double()
    w = torch.zeros((n, k))
    w[torch.arange(n), torch.arange(n) % k] = 1.0
    b = (torch.round((torch.randn(n, generator=g) * (0.8 * std) + mean) * s * 1024) / 1024).float()
    pre = x64[:, torch.arange(n) % k] + b.double()
    assert torch.equal(pre, pre.float().double())
    got = mbrt.mx_linear(xs, mbrt.mx_quantize(w.cuda()), b.cuda(), act=act, out_dtype=mbrt.MxTensor)
    torch.cuda.synchronize()
    want, bound = _gelu(pre, act)
    ref.check_held(got, want, bound, f"GELU {act} around {mean}")


AROUND = [(0.0, 1.0), (-3.0, 0.5), (-5.0, 0.3), (-6.5, 0.3), (-8.0, 0.2), (-11.0, 0.2), (-12.5, 0.4), (-30.0, 9.0)]


@pytest.mark.parametrize("mean,std", AROUND)
@pytest.mark.parametrize("act", [1, 2])
@pytest.mark.parametrize("x", [MX, BF16, F16, F32])
@pytest.mark.parametrize("rows,n", [(3, 16384), (64, 320), (700, 320)])
def test_tail_values(dev, rows, n, x, act, mean, std):
    """A few rows against many weights, strips, small tiles."""
    _run(rows, n, x, act, mean, std)


@pytest.mark.parametrize("mean,std", [(0.0, 1.0), (-5.0, 0.3), (-11.0, 0.2)])
@pytest.mark.parametrize("x,act", [(MX, 1), (MX, 2), (BF16, 2), (F16, 1)])
def test_tail_values_of_large_tiles(dev, x, act, mean, std):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    n = 1024
    rows = 128 * -(-(2 * cus if x == MX else cus // 2) // (n // 128)) + 5    # as many tiles of 128 x 128 as that form begins with
    _run(rows, n, x, act, mean, std)
