"""GPU tests of the norms around a block against their 64-bit form, with derived bounds (mx_ref.py)."""
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
EPS = 1e-12


def _rand(seed, shape, dtype=F32, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(dtype).cuda()


def _gate(kind, lead, D, dtype, seed=9):
    if kind is None:
        return None
    shape = dict(token=(*lead, 1), full=(*lead, D), batch=(lead[0], *[1] * (len(lead) - 1), D), one=(D,), scalar=(1,),
                 position=(*lead[1:], D), entry=(lead[0], *[1] * (len(lead) - 1), 1))[kind]
    return _rand(seed, shape, dtype)


def _verify(got, residual, update, gamma, post_gamma, gate, logit, ls, alpha, out, post_scale, scale, eps, before=None):
    """before: residual and update as they were, where the call wrote over them."""
    h, normed = got
    residual, update = before or (residual, update)
    want, bound = ref.block_sum(residual, update, post_gamma, gate, logit, ls, alpha, post_scale, eps)
    layer_ref.check(h, want, bound + layer_ref.half_step(residual.dtype, want), "sum")
    if gamma is None:
        assert normed is None
        return
    want, bound = ref.norm(h, gamma, scale, eps)   # of the sum as it is stored
    if out == MX:
        ref.check_held(normed, want, bound, "normed")
    else:
        layer_ref.check(normed, want, bound + layer_ref.half_step(out, want), "normed")


def _case(lead, D, rdt, udt, out, gate=None, gdt=None, logit=False, post=True, scaled=True, alpha=1.0, pre=True, seed=0, **kw):
    import mbrt

    say(f"block_norm {lead} D={D} {rdt} {udt} -> {out} gate={gate} logit={logit} post={post} scaled={scaled} alpha={alpha}")
    r, u = _rand(seed, (*lead, D), rdt, 2.0), _rand(seed + 1, (*lead, D), udt)
    gamma = _rand(seed + 2, (D,), F32, 0.1, 1.0) if pre else None
    pg = _rand(seed + 3, (D,), BF16, 0.1, 1.0) if post else None
    ls = _rand(seed + 4, (D,), F16, 0.1, 0.3) if scaled else None
    g = _gate(gate, lead, D, gdt or udt)
    got = mbrt.block_norm(r, u, gamma, post_gamma=pg, gate=g, gate_is_logit=logit, layer_scale=ls, alpha=alpha,
                          out_dtype=None if not pre else mbrt.MxTensor if out == MX else out, **kw)
    torch.cuda.synchronize()
    root = D ** 0.5
    _verify(got, r, u, gamma, pg, g, logit, ls, alpha, out, kw.get("post_scale", root), kw.get("scale", root), kw.get("eps", EPS))
    if pre:   # the same without the sum
        again = mbrt.block_norm(r, u, gamma, post_gamma=pg, gate=g, gate_is_logit=logit, layer_scale=ls, alpha=alpha,
                                out_dtype=mbrt.MxTensor if out == MX else out, store_sum=False, **kw)
        assert again[0] is None
        for a, b in zip(again[1] if out == MX else [again[1]], got[1] if out == MX else [got[1]]):
            assert torch.equal(torch.as_tensor(a), torch.as_tensor(b))


DIMS = [1, 2, 3, 5, 8, 20, 31, 33, 64, 127, 256, 257, 384, 500, 512, 767, 1001, 1536, 2049, 4096, 4100, 8192, 8200]


@pytest.mark.parametrize("rdt,udt,out", [(F32, F32, F32), (F32, BF16, BF16), (BF16, BF16, BF16), (F16, F16, MX), (BF16, F32, F16),
                                         (F32, F16, MX), (F16, BF16, F32)])
@pytest.mark.parametrize("D", DIMS)
def test_sizes_and_types(dev, D, rdt, udt, out):
    _case((3, 7), D, rdt, udt, out, seed=D)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 65, 1000])
def test_row_counts(dev, rows):
    _case((rows,), 384, BF16, BF16, BF16, seed=rows)
    _case((rows,), 1536, F32, BF16, MX, seed=rows)


@pytest.mark.parametrize("gate", ["token", "full", "batch", "one", "scalar", "position", "entry"])
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("D,rdt,udt,out,gdt", [(384, BF16, BF16, BF16, BF16), (129, F32, F32, MX, F32), (96, F16, F16, F16, F32),
                                               (4100, BF16, BF16, MX, F16), (3, F32, BF16, F32, BF16), (200, F32, F16, BF16, F16)])
def test_gates(dev, gate, logit, D, rdt, udt, out, gdt):
    _case((4, 9), D, rdt, udt, out, gate=gate, gdt=gdt, logit=logit, seed=D)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("D", [384, 77, 5])
def test_parts_left_out(dev, post, scaled, pre, D):
    _case((5, 8), D, F32, BF16, BF16, post=post, scaled=scaled, pre=pre, alpha=0.25, seed=3)
    if pre:
        _case((5, 8), D, BF16, F16, MX, gate="token", logit=True, post=post, scaled=scaled, seed=4, scale=1.5, post_scale=0.5, eps=1e-3)


@pytest.mark.parametrize("D", [96, 1001, 5000])
@pytest.mark.parametrize("rdt,udt", [(F32, BF16), (BF16, BF16)])
def test_in_place(dev, D, rdt, udt):
    import mbrt

    r, u, gamma = _rand(1, (50, D), rdt), _rand(2, (50, D), udt), _rand(3, (D,), F32, 0.1, 1.0)
    want = mbrt.block_norm(r, u, gamma, post_gamma=gamma, alpha=0.5)
    r1, u1 = r.clone(), u.clone()
    h, n = mbrt.block_norm(r1, u1, gamma, post_gamma=gamma, alpha=0.5, sum_out=r1, normed=u1)
    assert h is r1 and n is u1 and torch.equal(r1, want[0]) and torch.equal(u1, want[1])
    u2 = u.clone()
    assert torch.equal(mbrt.block_norm(r, u2, gamma, post_gamma=gamma, alpha=0.5, normed=u2, store_sum=False)[1], want[1])
    with pytest.raises(mbrt.MbrtError, match="overlaps"):
        mbrt.block_norm(r1, u1, gamma, normed=r1)
    with pytest.raises(mbrt.MbrtError, match="overlaps"):
        mbrt.block_norm(r1[:49], u1[:49], gamma, sum_out=r1[1:])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,pad,off", [(64, 8, 8), (64, 3, 1), (45, 5, 2), (9000, 7, 1)])
def test_strides_and_what_lies_around(dev, dtype, D, pad, off):
    import mbrt

    rows = 30
    say(f"strided block_norm D={D} pad={pad} off={off} {dtype}")

    def inside(seed, fill):
        big = torch.full((rows + 1, D + pad), fill, dtype=dtype, device="cuda")
        return big, big[:rows, off:off + D]

    (_, r), (_, u), (_, g) = (inside(i, math.nan) for i in range(3))
    for i, t in enumerate((r, u, g)):
        t.copy_(_rand(i, (rows, D), dtype))
    (sbig, s), (obig, o) = inside(4, 7.0), inside(5, 7.0)
    gamma = _rand(5, (D,), F32, 0.1, 1.0)
    got = mbrt.block_norm(r, u, gamma, post_gamma=gamma, gate=g, sum_out=s, normed=o)
    _verify(got, r, u, gamma, gamma, g, False, None, 1.0, dtype, D ** 0.5, D ** 0.5, EPS)
    for big in (sbig, obig):
        assert bool((big[rows] == 7).all() and (big[:, :off] == 7).all() and (big[:, off + D:] == 7).all())
    nb = -(-D // 32)
    codes = torch.full((rows + 1, 16 * nb + 32), 0x5A, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows + 1, nb + 3), 0x5A, dtype=torch.uint8, device="cuda")
    held = mbrt.MxTensor(codes[:rows, 16:16 + 16 * nb], scales[:rows, 1:1 + nb], D)
    got = mbrt.block_norm(r, u, gamma, post_gamma=gamma, gate=g, normed=held)
    _verify(got, r, u, gamma, gamma, g, False, None, 1.0, MX, D ** 0.5, D ** 0.5, EPS)
    assert bool((codes[:, :16] == 0x5A).all() and (codes[:, 16 + 16 * nb:] == 0x5A).all() and (codes[rows] == 0x5A).all())
    assert bool((scales[:, :1] == 0x5A).all() and (scales[:, 1 + nb:] == 0x5A).all() and (scales[rows] == 0x5A).all())


@pytest.mark.parametrize("D", [64, 45, 5000])
def test_specials(dev, D):
    """NaN and infinities stay in their row; a row of zeros is zeros."""
    import mbrt

    r, u, gamma = _rand(1, (6, D)), _rand(2, (6, D)), torch.ones(D, device="cuda")
    r[1, D - 1], u[2, D - 2] = math.nan, math.inf
    r[3], u[3] = 0, 0
    h, n = mbrt.block_norm(r, u, gamma, post_gamma=gamma)
    h64, _ = ref.block_sum(r, u, gamma, None, False, None, 1.0, D ** 0.5, EPS)
    n64, _ = ref.norm(h, gamma, D ** 0.5, EPS)
    assert torch.equal(torch.isnan(h.cpu()), torch.isnan(h64)) and torch.equal(torch.isnan(n.cpu()), torch.isnan(n64))
    assert bool((h[3] == 0).all() and (n[3] == 0).all())
    held = mbrt.block_norm(r, u, gamma, post_gamma=gamma, out_dtype=mbrt.MxTensor)[1]
    assert bool((held.scales[1] == 255).all() and (held.scales[2] == 255).all() and (held.scales[3] == 0).all())


def test_rows_far_apart(dev):
    import mbrt

    rows, D, stride = 70000, 40, 32768
    big = torch.empty(rows * stride, dtype=F32, device="cuda")
    r = big.as_strided((rows, D), (stride, 1))
    r.copy_(_rand(1, (rows, D)))
    u, gamma = _rand(2, (rows, D), BF16), _rand(3, (D,), F32, 0.1, 1.0)
    before = r.clone()
    got = mbrt.block_norm(r, u, gamma, sum_out=r)
    _verify(got, r, u, gamma, None, None, False, None, 1.0, BF16, 1.0, D ** 0.5, EPS, before=(before, u))


@pytest.mark.parametrize("D", [3, 8])
def test_more_rows_than_a_launch_has(dev, D):
    """The rows around 2^23, and the last ones, as in a call of their own."""
    import mbrt

    rows = (1 << 24) + 77
    g = torch.Generator(device="cuda").manual_seed(1)
    r, u = (torch.randn((rows, D), generator=g, device="cuda").to(BF16) for _ in range(2))
    gate = torch.randn((rows, 1), generator=g, device="cuda")
    gamma, post = _rand(3, (D,), F32, 0.1, 1.0), _rand(4, (D,), F32, 0.1, 1.0)
    h, n = mbrt.block_norm(r, u, gamma, post_gamma=post, gate=gate, gate_is_logit=True)
    held = mbrt.block_norm(r, u, gamma, gate=gate, store_sum=False, out_dtype=mbrt.MxTensor)[1]
    for a, b in ((0, 9), ((1 << 23) - 9, (1 << 23) + 9), (rows - 99, rows)):
        part = r[a:b], u[a:b], gamma
        h2, n2 = mbrt.block_norm(*part, post_gamma=post, gate=gate[a:b], gate_is_logit=True)
        held2 = mbrt.block_norm(*part, gate=gate[a:b], store_sum=False, out_dtype=mbrt.MxTensor)[1]
        assert torch.equal(h[a:b], h2) and torch.equal(n[a:b], n2)
        assert torch.equal(held.codes[a:b], held2.codes) and torch.equal(held.scales[a:b], held2.scales)


def test_captured_on_another_stream_and_without_the_extension_module(dev, monkeypatch):
    import mbrt
    from mbrt import _calls

    r, u, gamma, g = _rand(1, (2, 90, 384)), _rand(2, (2, 90, 384), BF16), _rand(3, (384,)), _rand(4, (2, 1, 384), BF16)
    call = lambda **kw: mbrt.block_norm(r, u, gamma, post_gamma=gamma, gate=g, gate_is_logit=True, alpha=0.5, **kw)
    want = call()
    held = call(out_dtype=mbrt.MxTensor)[1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = call(stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    h, n = torch.empty_like(r), torch.empty_like(u)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(sum_out=h, normed=n)
    for i in range(3):
        r.copy_(_rand(20 + i, (2, 90, 384)))
        h.zero_(), n.zero_()
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(h, eager[0]) and torch.equal(n, eager[1]), i
    r.copy_(_rand(1, (2, 90, 384)))
    monkeypatch.setattr(mbrt, "_n", _calls)
    got = call()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    again = call(out_dtype=mbrt.MxTensor)[1]
    assert torch.equal(again.codes, held.codes) and torch.equal(again.scales, held.scales)
