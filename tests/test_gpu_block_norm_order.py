"""GPU tests of the norms around a block against the formula in torch's f32 operations on the same device (whose square root is
within a step, not correctly rounded): where the sums of squares are exact in any order, every result is the formula's, bit for
bit; where they are not, a stored sum of 2 bytes falls to another side than in 64 bits no more often than the formula's does."""
from __future__ import annotations

import pytest
import torch

from gpu_util import say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-12


def _rand(seed, shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype).cuda()


def _whole(seed, shape, dtype):
    return torch.randint(-8, 9, shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _rms(t, gamma, scale, eps):
    # squares up to 2^6 of 2^14 features at most: the sum is a whole number below 2^24, exact in any order
    return t * (scale * gamma.float()) / torch.sqrt((t * t).sum(-1, keepdim=True) + eps)


def _scale(D):
    return float(torch.tensor(D ** 0.5, dtype=F32))


# a few lanes to a row, a wave, a block, element by element; whole chunks and cut ones
DIMS = [2, 96, 384, 385, 512, 700, 767, 1001, 1536, 2048, 4100, 8192, 9001]


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("rdt,udt,gdt", [(F32, F32, F32), (F32, BF16, BF16), (BF16, BF16, BF16), (F16, F16, F16), (BF16, F16, F32)])
def test_sum_bit_for_bit(dev, D, rdt, udt, gdt):
    import mbrt

    say(f"block_norm order D={D} {rdt} {udt}")
    r, u, gate = _rand(1, (9, 40, D), rdt, 2.0), _whole(2, (9, 40, D), udt), _rand(3, (9, 1, D), gdt)
    post, ls = _rand(4, (D,), F32, 0.1, 1.0), _rand(5, (D,), F32, 0.05, 0.3)
    for alpha, g, s in ((1.0, gate, ls), (0.5, None, ls), (1.0, gate, None)):
        want = _rms(u.float(), post, _scale(D), EPS)
        if s is not None:
            want = want * s
        if g is not None:
            want = want * g.float()
        want = (r.float() + alpha * want).to(rdt)
        got, none = mbrt.block_norm(r, u, post_gamma=post, gate=g, layer_scale=s, alpha=alpha, eps=EPS)
        assert none is None and torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("rdt,udt,out", [(F32, F32, F32), (F32, BF16, BF16), (BF16, BF16, F32), (F16, F16, F16), (BF16, BF16, BF16)])
def test_normed_bit_for_bit(dev, D, rdt, udt, out):
    import mbrt

    say(f"block_norm order normed D={D} {rdt} -> {out}")
    r, u = _whole(1, (9, 40, D), rdt) / 2, _whole(2, (9, 40, D), udt) / 2   # their sum has steps of a half up to 8
    gamma = _rand(4, (D,), F32, 0.1, 1.0)
    h = r.float() + u.float()
    want = _rms(h, gamma, _scale(D), EPS)
    got, normed = mbrt.block_norm(r, u, gamma, eps=EPS, out_dtype=out)
    assert torch.equal(got, h.to(rdt))
    assert torch.equal(normed, want.to(out)), int((normed != want.to(out)).sum())
    held = mbrt.block_norm(r, u, gamma, eps=EPS, out_dtype=mbrt.MxTensor, store_sum=False)[1]
    same = mbrt.mx_quantize(want)
    assert torch.equal(held.codes, same.codes) and torch.equal(held.scales, same.scales)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,D", [(24000, 384), (6000, 1536)])
def test_sides_of_a_rounding(dev, dtype, rows, D):
    """Sums of 2 bytes whose f32 value lies on a tie fall to either side; against 64 bits as often as the formula's in f32."""
    import mbrt

    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda shape: torch.randn(shape, generator=g, device="cuda")
    r, u = (rand((rows, D)) * 2).to(dtype), rand((rows, D)).to(dtype)
    post = rand((D,)) * 0.1 + 1
    h = mbrt.block_norm(r, u, post_gamma=post, eps=EPS)[0]
    uf = u.float()
    plain = (r.float() + uf * (_scale(D) * post) / torch.sqrt((uf * uf).sum(-1, keepdim=True) + EPS)).to(dtype)
    ud = u.double()
    exact = (r.double() + ud * (D ** 0.5 * post.double()) / torch.sqrt((ud * ud).sum(-1, keepdim=True) + EPS)).to(dtype)
    ours, theirs, apart = (int((a != b).sum()) for a, b in ((h, exact), (plain, exact), (h, plain)))
    say(f"sides {dtype} [{rows}, {D}]: {ours}, the formula in f32 {theirs}, apart {apart}")
    # independent counts of some hundred: half as many again is many deviations away
    assert theirs > 100 and ours <= 1.5 * theirs and apart <= theirs
