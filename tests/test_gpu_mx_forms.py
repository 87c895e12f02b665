"""GPU tests of the forms that only large calls of the 4-bit layer and the norms around a block take, with row counts derived
from the device's compute units, so that the forms stay covered; and of the largest and smallest scales."""
from __future__ import annotations

import pytest
import torch

import layer_ref
import mx_ref as ref
from gpu_util import say
from test_gpu_block_norm import _case as norm_case
from test_gpu_mx_linear import BF16, F16, F32, MX, _case, _operand, _rand

pytestmark = pytest.mark.gpu


def _cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _rows(tiles, n):
    """Rows for this many tiles of 128 x 128, and some of another row of tiles."""
    return 128 * -(-tiles // -(-n // 128)) + 37


@pytest.mark.parametrize("act,bias,res", [(0, F32, None), (0, None, BF16), (1, BF16, None), (2, F32, None), (2, F16, F32), (3, BF16, F16), (4, F16, None)])
@pytest.mark.parametrize("k,n", [(200, 1031), (544, 1152)])
def test_both_sides_in_4_bits_in_large_tiles(dev, k, n, act, bias, res):
    """128 x 128 tiles from two for every compute unit on; 7 and 17 blocks of K, so that a group of 16 scales is cut."""
    _case(dev, _rows(2 * _cus(), n), k, n, MX, MX, act=act, bias=bias, res=res, seed=act)


@pytest.mark.parametrize("act", [1, 2, 3, 4])
@pytest.mark.parametrize("x,out,bias,res", [(MX, BF16, F16, None), (MX, F32, BF16, F32), (MX, F16, F32, F16), (BF16, BF16, F16, BF16), (BF16, F32, F32, None),
                                            (F16, F16, BF16, None), (F16, F32, F16, F32), (BF16, MX, BF16, None), (F16, MX, F16, F32)])
def test_activations_in_large_tiles(dev, x, out, bias, res, act):
    """128 x 128 tiles from one for every compute unit on for x in 4 bits, from half as many for x in 16."""
    n = 523
    _case(dev, _rows(_cus() if x == MX else -(-_cus() // 2), n), 136, n, x, out, act=act, bias=bias, res=res, seed=act)


@pytest.mark.parametrize("act", [1, 2, 3, 4])
@pytest.mark.parametrize("out,res", [(BF16, None), (F32, F32)])
def test_activations_of_long_k(dev, out, res, act):
    """256 x 256 tiles: 48 blocks of K and more, four fifths of a round of the compute units."""
    _case(dev, 256 * -(-_cus() // 4) - 3, 1538, 1021, MX, out, act=act, bias=F16, res=res, seed=act)


@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("x", [MX, BF16, F16, F32])
@pytest.mark.parametrize("rows,k,n", [(3, 70, 8200), (40, 70, 90), (700, 70, 300)])
def test_activations_in_4_bits(dev, rows, k, n, x, act):
    _case(dev, rows, k, n, x, MX, act=act, bias=F16, seed=act)
    _case(dev, rows, k, n, x, MX, act=act, bias=None, res=BF16, seed=act + 10)


# ---- norms: three chunks to a lane of a wave, 129 to 192 of them in a row, from 16 rows for every compute unit on -----

@pytest.mark.parametrize("D,rdt,udt,out", [(513, F32, F32, F32), (640, F32, BF16, BF16), (767, BF16, F32, F16), (768, F32, F16, MX), (700, F16, F16, F32),
                                           (1025, BF16, BF16, BF16), (1111, F16, F16, MX), (1300, F16, F16, F16), (1536, BF16, BF16, BF16), (1536, BF16, BF16, MX)])
def test_three_chunks_to_a_lane(dev, D, rdt, udt, out):
    rows = 16 * _cus()
    norm_case((rows + 5,), D, rdt, udt, out, gate="token", logit=True, alpha=0.5, seed=D)
    norm_case((5, rows // 4), D, rdt, udt, out, gate="batch", post=False, scaled=False, seed=D + 1)


@pytest.mark.parametrize("D,dtype", [(767, F32), (700, F32), (1535, BF16), (1536, F16)])
def test_three_chunks_to_a_lane_in_place(dev, D, dtype):
    import mbrt

    rows = 16 * _cus() + 3
    say(f"block_norm in place rows={rows} D={D} {dtype}")
    r, u, gamma = _rand(1, (rows, D), dtype), _rand(2, (rows, D), dtype), _rand(3, (D,), F32)
    want = mbrt.block_norm(r, u, gamma, post_gamma=gamma, alpha=0.5)
    h, n = mbrt.block_norm(r, u, gamma, post_gamma=gamma, alpha=0.5, sum_out=r, normed=u)
    assert h is r and n is u and torch.equal(r, want[0]) and torch.equal(u, want[1])


# ---- scales at their ends ---------------------------------------------------------------------------

def _weights(n, blocks, byte, top, seed):
    """Rows of blocks under one scale byte, with codes 0 .. top of either sign; their values in 64 bits."""
    import mbrt

    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, top + 1, (n, 32 * blocks), generator=g) + 8 * torch.randint(0, 2, (n, 32 * blocks), generator=g)
    w = mbrt.MxTensor((c[:, 0::2] | c[:, 1::2] << 4).to(torch.uint8).cuda(), torch.full((n, blocks), byte, dtype=torch.uint8, device="cuda"), 32 * blocks)
    return w, ref.values(c, torch.full((n, blocks), byte), 32 * blocks)


@pytest.mark.parametrize("x", [MX, BF16, F16, F32])
@pytest.mark.parametrize("byte,top,e", [(0, 7, 60), (1, 7, 60), (252, 7, -60), (253, 5, -60), (254, 3, -60), (253, 7, -60), (254, 7, -60)])
@pytest.mark.parametrize("rows,n", [(3, 8200), (20, 40), (300, 200)])
def test_weights_under_the_smallest_and_largest_scales(dev, rows, n, x, byte, top, e):
    """x of a size that leaves the products f32's normal numbers (f16, which is not that wide, meets scale bytes 20 and 21).  A weight of 2^128 or more (codes 6 and 7 under byte 253, 4 to 7
    under 254) is beyond bf16: with x in 16 or 32 bits its output feature is not finite; with x in 4 bits it counts as it is."""
    import mbrt

    say(f"scale byte {byte} top {top} rows={rows} n={n} x={x}")
    if x == F16:
        byte, e = (byte + 20, 10) if byte < 2 else (byte, -20)
    w, w64 = _weights(n, 2, byte, top, 3)
    v = _rand(1, (rows, 64), F32).double().cpu()
    v = torch.where(v == 0, torch.ones_like(v), v) * 2.0 ** e
    xs = mbrt.mx_quantize(v.float().cuda()) if x == MX else v.to(x).cuda()
    x64 = ref.held(xs) if x == MX else xs.cpu().double()
    got = mbrt.mx_linear(xs, w, out_dtype=F32)
    want, bound = ref.linear(x64, w64, None, 0, None, F32)
    if x != MX:
        beyond = (w64.abs() >= 2.0 ** 128).any(-1)
        assert bool(beyond.any()) == ((byte, top) in ((253, 7), (254, 7)))
        assert not bool(torch.isfinite(got.cpu()[:, beyond]).any())
        got, want, bound = got[:, (~beyond).cuda()], want[:, ~beyond], bound[:, ~beyond]
    layer_ref.check(got, want, bound, f"scale byte {byte}")
