"""GPU tests of the qkv split with head norms and rotation against its 64-bit form."""
from __future__ import annotations

import math

import pytest
import torch

import layer_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(seed, shape, dtype, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(dtype).cuda()


def _tables(n_pos, D, dtype=F32):
    ang = torch.arange(n_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return torch.cos(ang).to(dtype).cuda(), torch.sin(ang).to(dtype).cuda()


def _heads(B, H, N, D, dtype, order):
    if order == "bhnd":
        return torch.full((B, H, N, D), 7.0, dtype=dtype, device="cuda")
    return torch.full((B, N, H, D), 7.0, dtype=dtype, device="cuda").permute(0, 2, 1, 3)


def _case(B, N, H, KV, D, dtype, out_dtype=None, order="bnhd", pos0=0, gamma=F32, trig=F32, scale=None, eps=1e-12,
          with_v=True, std=1.0):
    import mbrt

    out_dtype = out_dtype or dtype
    say(f"qkv norm B={B} N={N} H={H} KV={KV} D={D} {dtype} -> {out_dtype} {order} pos0={pos0} v={with_v}")
    qkv = _rand(B + N, (B, N, (H + 2 * KV) * D), dtype, std)
    qg, kg = _rand(1, (D,), gamma, 0.2, 1.0), _rand(2, (D,), gamma, 0.2, 1.0)
    cos, sin = _tables(pos0 + N + 3, D, trig)
    q, k, v = (_heads(B, h, N, D, out_dtype, order) for h in (H, KV, KV))
    mbrt.split_qkv_norm_rotary(qkv, qg, kg, cos, sin, q, k, v if with_v else None, H, kv_heads=KV, scale=scale, eps=eps,
                               pos0=pos0)
    torch.cuda.synchronize()
    want = ref.qkv_norm(qkv, qg, kg, cos, sin, H, KV, math.sqrt(D) if scale is None else scale, eps, pos0, out_dtype)
    for got, (y, bound), name in zip((q, k, v), want, "qkv"):
        if name == "v" and not with_v:
            assert bool((v == 7).all())
        else:
            ref.check(got, y, bound, name)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [2, 6, 8, 16, 32, 48, 64, 96, 128, 192, 256, 512, 600])
def test_head_sizes(dev, D, dtype):
    _case(2, 5, 3, 3, D, dtype)
    _case(1, 7, 4, 1, D, dtype, order="bhnd", pos0=11)


@pytest.mark.parametrize("B,N,H,KV", [(1, 1, 1, 1), (60, 1, 8, 8), (3, 33, 8, 2), (1, 257, 6, 3), (5, 4, 1, 1), (2, 3, 33, 11)])
@pytest.mark.parametrize("with_v", [True, False])
def test_head_counts(dev, B, N, H, KV, with_v):
    _case(B, N, H, KV, 64, BF16, with_v=with_v)
    _case(B, N, H, KV, 64, F32, with_v=with_v, order="bhnd")


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F32, BF16), (F16, BF16), (F32, F16)])
@pytest.mark.parametrize("gamma,trig", [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
def test_types(dev, dtype, out, gamma, trig):
    _case(2, 9, 4, 2, 64, dtype, out, gamma=gamma, trig=trig)
    _case(2, 9, 4, 2, 10, dtype, out, gamma=gamma, trig=trig)


def test_scale_eps_small_and_large_values(dev):
    _case(1, 4, 2, 2, 64, F32, scale=3.0, eps=0.5)
    _case(1, 4, 2, 2, 64, F32, std=1e-6, eps=1e-6)
    _case(1, 4, 2, 2, 64, BF16, std=1e4)


def test_zero_vectors_and_specials_stay_in_their_head(dev):
    import mbrt

    qkv = _rand(1, (1, 4, 6 * 64), F32)
    qkv[0, 0, :64] = 0.0
    qkv[0, 1, 64] = float("nan")       # head 1 of q
    qkv[0, 2, 128] = float("inf")      # head 0 of k
    g = torch.ones(64, device="cuda")
    cos, sin = _tables(4, 64)
    q, k, v = (_heads(1, 2, 4, 64, F32, "bhnd") for _ in range(3))
    mbrt.split_qkv_norm_rotary(qkv, g, g, cos, sin, q, k, v, 2)
    assert bool((q[0, 0, 0] == 0).all())
    bad = torch.isnan(q).any(-1)[0]
    assert bad.nonzero().tolist() == [[1, 1]]
    assert (~torch.isfinite(k)).any(-1)[0].nonzero().tolist() == [[0, 2]]


@pytest.mark.parametrize("dtype,D,off", [(BF16, 64, 0), (BF16, 64, 1), (F32, 64, 3), (F16, 12, 0)])
def test_strided_input_and_cache_rows(dev, dtype, D, off):
    """qkv inside wider rows, keys and values straight into their rows of a longer cache."""
    import mbrt

    B, N, H, KV, cap, at = 2, 3, 4, 2, 20, 9
    width = (H + 2 * KV) * D
    wide = torch.full((B, N, width + 16), float("nan"), dtype=dtype, device="cuda")
    qkv = wide[:, :, off:off + width]
    qkv.copy_(_rand(1, (B, N, width), dtype))
    cache = torch.full((2, B, cap, KV, D), 7.0, dtype=dtype, device="cuda")
    kc, vc = (cache[i, :, at:at + N].permute(0, 2, 1, 3) for i in range(2))
    q = _heads(B, H, N, D, dtype, "bnhd")
    g = _rand(3, (D,), F32, 0.2, 1.0)
    cos, sin = _tables(at + N, D)
    mbrt.split_qkv_norm_rotary(qkv, g, g, cos, sin, q, kc, vc, H, kv_heads=KV, pos0=at)
    want = ref.qkv_norm(qkv, g, g, cos, sin, H, KV, math.sqrt(D), 1e-12, at, dtype)
    for got, (y, bound) in zip((q, kc, vc), want):
        ref.check(got, y, bound, "cache")
    assert bool((cache[:, :, :at] == 7).all() and (cache[:, :, at + N:] == 7).all())


@pytest.mark.parametrize("D", [64, 10])
def test_in_place(dev, D):
    """q and k normed and rotated where they stand in the projection."""
    import mbrt

    B, N, H, KV = 3, 40, 8, 2
    qkv = _rand(1, (B, N, (H + 2 * KV) * D), BF16)
    before = qkv.clone()
    g = _rand(3, (D,), F32, 0.2, 1.0)
    cos, sin = _tables(N, D)
    heads = qkv.view(B, N, H + 2 * KV, D).permute(0, 2, 1, 3)
    mbrt.split_qkv_norm_rotary(qkv, g, g, cos, sin, heads[:, :H], heads[:, H:H + KV], None, H, kv_heads=KV)
    want = ref.qkv_norm(before, g, g, cos, sin, H, KV, math.sqrt(D), 1e-12, 0, BF16)
    ref.check(heads[:, :H], *want[0], "q")
    ref.check(heads[:, H:H + KV], *want[1], "k")
    assert torch.equal(qkv[..., (H + KV) * D:], before[..., (H + KV) * D:])


def test_agrees_with_norm_then_rotary_calls(dev):
    """The same heads through the library's norm and rotary calls: f32 throughout, a few steps apart."""
    import mbrt

    B, N, H, D = 2, 50, 4, 64
    qkv = _rand(1, (B, N, 3 * H * D), F32)
    g = _rand(2, (D,), F32, 0.2, 1.0)
    cos, sin = _tables(N, D)
    q, k, v = (_heads(B, H, N, D, F32, "bhnd") for _ in range(3))
    mbrt.split_qkv_norm_rotary(qkv, g, g, cos, sin, q, k, v, H)
    part = qkv.view(B, N, 3, H, D).permute(2, 0, 3, 1, 4).contiguous()
    normed = torch.empty_like(part[0])
    mbrt.rms_norm(part[0], g, normed, math.sqrt(D))
    mbrt.rotary_(normed.view(B * H, N, D), None, cos, sin)
    pair = normed.double().view(B, H, N, D // 2, 2).norm(dim=-1).repeat_interleave(2, -1)
    # each side within (D / 2 + 8) U of the pair's terms, at most sqrt(2) times its norm
    assert bool(((q.double() - normed.double()).abs() <= 2 * 1.5 * (D / 2 + 8) * ref.U * pair).all())
    assert torch.equal(v, part[2])


def test_captured_and_on_another_stream(dev):
    import mbrt

    B, N, H, D = 2, 30, 8, 64
    qkv = _rand(1, (B, N, 3 * H * D), BF16)
    g = _rand(2, (D,), F32, 0.2, 1.0)
    cos, sin = _tables(N, D)
    outs = [[_heads(B, H, N, D, BF16, "bnhd") for _ in range(3)] for _ in range(3)]
    mbrt.split_qkv_norm_rotary(qkv, g, g, cos, sin, *outs[0], H)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    mbrt.split_qkv_norm_rotary(qkv, g, g, cos, sin, *outs[1], H, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mbrt.split_qkv_norm_rotary(qkv, g, g, cos, sin, *outs[2], H)
    for _ in range(3):
        for t in outs[2]:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(*outs):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("path", ["native", "ctypes"])
def test_strides_that_nothing_uses(dev, path, monkeypatch):
    """Strides of dimensions of size 1 may be anything, and differ between keys and values."""
    import mbrt
    from mbrt import _calls

    if path == "ctypes":
        monkeypatch.setattr(mbrt, "_n", _calls)
    for B, N, H, KV in ((1, 20, 2, 2), (3, 1, 2, 1), (1, 1, 1, 1)):
        say(f"single indices B={B} N={N} {H}/{KV}")
        qkv = _rand(1, (B, N, (H + 2 * KV) * 64), BF16)
        gamma, (cos, sin) = torch.ones(64, device="cuda"), _tables(N, 64)
        outs = []
        for odd in (False, True):
            views = []
            for i, h in enumerate((H, KV, KV)):
                t = _heads(B, h, N, 64, BF16, "bhnd")
                st = [8 * t.numel() + 3 + i if odd and n == 1 else s for s, n in zip(t.stride(), t.shape)]
                views.append(t.as_strided(t.shape, st))
            mbrt.split_qkv_norm_rotary(qkv, gamma, gamma, cos, sin, *views, H, kv_heads=KV)
            outs.append([t.clone() for t in views])
        for a, b in zip(*outs):
            assert torch.equal(a, b)
