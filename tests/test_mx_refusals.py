"""CPU tests: what the 4-bit entry points and block_norm refuse, at the C-ABI and in the binding, before any launch.
Non-NULL pointers are stand-in addresses that are never read."""
from __future__ import annotations

import pytest

P = [(k + 1) << 32 for k in range(12)]
F32, F16, I64, BF16, I32, MX = 0, 1, 2, 3, 4, 5
OK, ARG, DTYPE, SHAPE, ALIGN = 0, 1, 2, 3, 4


@pytest.fixture(scope="module")
def lib():
    import mbrt

    if not mbrt.LIB_PATH.exists():
        pytest.skip("libmbrt.so not built")
    return mbrt.lib()


def _err(lib):
    return lib.mbrt_last_error().decode()


def test_quantize_arguments(lib):
    def call(x=P[0], dt=BF16, xs=64, c=P[1], cs=32, s=P[2], ss=2, rows=10, n=64):
        return lib.mbrt_mx_quantize(x, dt, xs, c, cs, s, ss, rows, n, None)

    def back(c=P[1], cs=32, s=P[2], ss=2, out=P[0], dt=BF16, os=64, rows=10, n=64):
        return lib.mbrt_mx_dequantize(c, cs, s, ss, out, dt, os, rows, n, None)

    for f in (call, back):
        assert f(dt=I64) == DTYPE and f(dt=MX) == DTYPE
        assert f(rows=-1) == SHAPE and f(n=-1) == SHAPE and f(n=1 << 28) == SHAPE and f(rows=1 << 40) == SHAPE
        assert f(c=None) == ARG and f(s=None) == ARG and "NULL" in _err(lib)
        assert f(c=P[1] + 8) == ALIGN and f(cs=40) == ALIGN and "16 bytes" in _err(lib)
        assert f(rows=0) == OK and f(n=0) == OK
    assert call(x=None) == ARG and call(x=P[0] + 1) == ALIGN and call(xs=-1) == SHAPE
    assert call(cs=16) == SHAPE and call(ss=1) == SHAPE and "overlap" in _err(lib)
    assert back(out=None) == ARG and back(out=P[0] + 1) == ALIGN and back(os=63) == SHAPE and back(cs=-16) == SHAPE and back(ss=-1) == SHAPE
    for kw in (dict(c=P[0]), dict(s=P[0] + 1279), dict(s=P[1] + 319), dict(c=P[0] + 1264)):
        assert call(**kw) == ARG and "overlaps" in _err(lib)
    for kw in (dict(out=P[1] + 318), dict(out=P[2] - 1278)):
        assert back(**kw) == ARG and "overlaps" in _err(lib)


def test_linear_arguments(lib):
    def call(x=P[0], dt=MX, xs=32, xsc=P[1], xss=2, w=P[2], ws=32, wsc=P[3], wss=2, b=None, bdt=F32, r=None, rdt=F32, rs=32, out=P[4],
             odt=BF16, os=32, osc=P[5], oss=1, rows=10, k=64, n=32, act=0):
        return lib.mbrt_mx_linear(x, dt, xs, xsc, xss, w, ws, wsc, wss, b, bdt, r, rdt, rs, out, odt, os, osc, oss, rows, k, n, act, None)

    assert call(dt=I64) == DTYPE and call(odt=I32) == DTYPE and call(b=P[6], bdt=MX) == DTYPE and call(r=P[6], rdt=I64) == DTYPE
    assert call(dt=6) == DTYPE and call(act=5) == ARG and call(act=-1) == ARG and "activation" in _err(lib)
    for kw in (dict(rows=-1), dict(k=-1), dict(n=-1), dict(k=1 << 28), dict(n=1 << 28, os=1 << 28), dict(rows=1 << 40), dict(xs=-16),
               dict(ws=-16), dict(xss=-1), dict(wss=-1), dict(r=P[6], rs=-1), dict(os=31), dict(odt=MX, os=0), dict(odt=MX, os=16, oss=0)):
        assert call(**kw) == SHAPE, kw
    for name in ("x", "xsc", "w", "wsc", "out"):
        assert call(**{name: None}) == ARG and "NULL" in _err(lib)
    assert call(odt=MX, os=16, osc=None) == ARG
    for kw in (dict(x=P[0] + 8), dict(xs=40), dict(w=P[2] + 8), dict(ws=40), dict(out=P[4] + 1), dict(odt=MX, os=16, out=P[4] + 8),
               dict(odt=MX, os=24), dict(b=P[6] + 2), dict(r=P[6] + 1, rdt=BF16), dict(dt=F32, x=P[0] + 2, xs=64)):
        assert call(**kw) == ALIGN, kw
    assert call(rows=0) == OK and call(n=0) == OK
    # an output within an operand
    for kw in (dict(out=P[0]), dict(out=P[0] + 318), dict(out=P[1] - 638), dict(out=P[2] + 1022), dict(out=P[3]), dict(b=P[6], out=P[6] + 126),
               dict(r=P[6], rdt=F32, out=P[6]), dict(r=P[6], rdt=BF16, rs=33, out=P[6]), dict(odt=MX, os=16, osc=P[4] + 159),
               dict(odt=MX, os=16, osc=P[0]), dict(odt=MX, os=16, osc=P[3] + 63), dict(odt=MX, os=16, r=P[4], rs=32)):
        assert call(**kw) == ARG and "overlaps" in _err(lib), kw


def test_linear_too_large_for_one_launch(lib):
    far = [(k + 1) << 50 for k in range(6)]
    for dt, rows, k, n in ((MX, 1 << 33, 64, 64), (BF16, 1 << 33, 64, 8), (F32, 1 << 33, 64, 64), (F16, 1 << 32, 64, 1000), (MX, 1 << 36, 0, 64)):
        assert lib.mbrt_mx_linear(far[0], dt, 0, far[1], 0, far[2], 32, far[3], 2, None, F32, None, F32, 0, far[4], BF16, n, None, 0,
                                  rows, k, n, 0, None) == SHAPE
        assert "too many" in _err(lib)


def test_block_norm_arguments(lib):
    def call(r=P[0], rdt=BF16, rs=64, u=P[1], udt=BF16, us=64, pg=None, pdt=F32, gate=None, gdt=BF16, gc=64, gs=64, gi=1, gp=10, logit=0,
             ls=None, ldt=F32, g=P[3], gad=F32, sum=P[4], ss=64, out=P[5], odt=BF16, os=64, osc=None, oss=0, rows=10, dim=64):
        return lib.mbrt_block_norm(r, rdt, rs, u, udt, us, pg, pdt, gate, gdt, gc, gs, gi, gp, logit, ls, ldt, g, gad, sum, ss, out, odt, os,
                                   osc, oss, rows, dim, 1.0, 8.0, 8.0, 1e-12, None)

    mx = dict(odt=MX, os=32, osc=P[6], oss=2)
    for kw in (dict(rdt=I64), dict(rdt=MX), dict(udt=MX), dict(odt=I32), dict(pg=P[7], pdt=I64), dict(gate=P[7], gdt=MX), dict(ls=P[7], ldt=4),
               dict(gad=I64)):
        assert call(**kw) == DTYPE, kw
    for kw in (dict(rows=-1), dict(rows=1 << 31), dict(dim=0), dict(dim=1 << 28), dict(rs=-1), dict(us=-1), dict(ss=63), dict(os=63),
               {**mx, "os": 16}, {**mx, "oss": 1}, dict(gate=P[7], gc=2), dict(gate=P[7], gi=0), dict(gate=P[7], gp=0), dict(gate=P[7], gs=-1)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(r=None), dict(u=None), dict(out=None), dict(g=None, out=None, sum=None), {**mx, "osc": None}):
        assert call(**kw) == ARG and "NULL" in _err(lib), kw
    for kw in (dict(r=P[0] + 1), dict(u=P[1] + 1), dict(sum=P[4] + 1), dict(out=P[5] + 1), {**mx, "out": P[5] + 8}, {**mx, "os": 40},
               dict(gate=P[7] + 1), dict(g=P[3] + 2), dict(pg=P[7] + 2), dict(ls=P[7] + 2)):
        assert call(**kw) == ALIGN, kw
    assert call(rows=0) == OK
    for kw in (dict(sum=P[0] + 2), dict(sum=P[0], ss=65), dict(sum=P[1]), dict(out=P[0]), dict(out=P[1] + 2), dict(out=P[1], odt=F32),
               dict(out=P[4]), dict(gate=P[4]), dict(gate=P[5], gp=1), dict(sum=P[3] + 254), dict(pg=P[5] + 1276), dict(ls=P[4]),
               {**mx, "out": P[1]}, {**mx, "osc": P[0]}, {**mx, "osc": P[5] + 319}, {**mx, "osc": P[4] + 1279}):
        assert call(**kw) == ARG and "overlaps" in _err(lib), kw


def test_binding_refusals(lib):
    import torch

    import mbrt

    E, u8 = torch.empty, torch.uint8
    x, bf = E(6, 70), torch.bfloat16
    held = lambda *s: mbrt.mx_empty(s, device="cpu")
    hx, w, out = held(6, 70), held(40, 70), E(6, 40, dtype=bf)
    q = lambda *a, **k: (lambda: mbrt.mx_quantize(*a, stream=0, **k))
    d = lambda *a, **k: (lambda: mbrt.mx_dequantize(*a, stream=0, **k))
    lin = lambda *a, **k: (lambda: mbrt.mx_linear(*a, stream=0, **k))
    bn = lambda *a, **k: (lambda: mbrt.block_norm(*a, stream=0, **k))
    r, g = E(2, 3, 8), E(8)
    for exc, match, fn in [
        (ValueError, r"codes \[", q(x, mbrt.MxTensor(hx.codes[:5], hx.scales, 70))),
        (ValueError, r"codes \[", q(x, mbrt.MxTensor(hx.codes, hx.scales[:, :2], 70))),
        (ValueError, r"x \[\.\., n\]", q(x, held(6, 71))),
        (TypeError, "uint8", q(x, mbrt.MxTensor(hx.codes.view(torch.int8), hx.scales, 70))),
        (TypeError, "torch.bool", q(x.bool(), hx)),
        (ValueError, "contiguous last dim", q(E(70, 6).t(), hx)),
        (ValueError, "more than one stride", q(E(4, 3, 8)[:, :2], held(4, 2, 8))),
        (ValueError, "one GPU", q(x, hx)),
        (ValueError, r"out \[\.\., n\]", d(hx, E(6, 64))),
        (ValueError, r"codes \[", d(hx, E(5, 70))),
        (ValueError, "disagree", d(hx, x, out_dtype=bf)),
        (ValueError, "one GPU", d(hx, x)),
        (TypeError, "MxTensor", lin(x, x, out=out)),
        (TypeError, "MxTensor", lin(1, w, out=out)),
        (ValueError, r"\[N, K\]", lin(x[:, :69], w, out=out)),
        (ValueError, r"\[N, K\]", lin(held(6, 64), w, out=out)),
        (ValueError, r"\[N, K\]", lin(x, held(2, 40, 70), out=out)),
        (ValueError, r"out and residual", lin(hx, w, out=out[:5])),
        (ValueError, r"out and residual", lin(hx, w, out=out, residual=out[:, :39])),
        (ValueError, r"out and residual", lin(hx, w, out=held(6, 41))),
        (ValueError, r"codes \[", lin(hx, w, out=held(5, 40))),
        (ValueError, r"codes \[", lin(mbrt.MxTensor(hx.codes, hx.scales[:5], 70), w, out=out)),
        (ValueError, r"bias \[N\]", lin(hx, w, E(39), out)),
        (ValueError, "disagree", lin(hx, w, out=out, out_dtype=torch.half)),
        (ValueError, "disagree", lin(hx, w, out=out, out_dtype=mbrt.MxTensor)),
        (ValueError, "disagree", lin(hx, w, out=held(6, 40), out_dtype=bf)),
        (ValueError, "contiguous last dim", lin(hx, w, out=E(40, 6).t())),
        (ValueError, "more than one stride", lin(held(3, 2, 70), w, out=E(3, 5, 40)[:, :2])),
        (TypeError, "torch.bool", lin(x.bool(), w, out=out)),
        (ValueError, "one GPU", lin(hx, w, out=out)),
        (TypeError, "Tensor", bn(r, 1, g)),
        (ValueError, "without gamma", bn(r, r, store_sum=False, sum_out=None)),
        (ValueError, "without gamma", bn(r, r, normed=r)),
        (ValueError, "disagree", bn(r, r, g, sum_out=r, store_sum=False)),
        (ValueError, "disagree", bn(r, r, g, sum_out=r, normed=E(2, 3, 8), out_dtype=bf)),
        (ValueError, "disagree", bn(r, r, g, sum_out=r, normed=held(2, 3, 8), out_dtype=bf)),
        (ValueError, r"\[\.\., D\]", bn(r, r[:1], g, sum_out=r, normed=r)),
        (ValueError, r"\[\.\., D\]", bn(r, r, g, sum_out=r[..., :7], normed=r)),
        (ValueError, r"\[\.\., D\]", bn(r, r, g, sum_out=r, normed=held(2, 3, 9))),
        (ValueError, "dtype", bn(r, r, g, sum_out=r.half(), normed=r)),
        (ValueError, r"gammas and layer_scale", bn(r, r, g[:7], sum_out=r, normed=r)),
        (ValueError, r"gammas and layer_scale", bn(r, r, g, layer_scale=E(1, 8), sum_out=r, normed=r)),
        (ValueError, "contiguous", bn(r, r, E(16)[::2], sum_out=r, normed=r)),
        (ValueError, "contiguous last dim", bn(E(2, 8, 3).transpose(1, 2), r, g, sum_out=r, normed=r)),
        (ValueError, "gate", bn(r, r, g, gate=E(2, 3, 4), sum_out=r, normed=r)),
        (ValueError, "gate", bn(r, r, g, gate=E(3, 3, 8), sum_out=r, normed=r)),
        (ValueError, "gate", bn(r, r, g, gate=E(1, 2, 3, 8), sum_out=r, normed=r)),
        (ValueError, "gate", bn(r, r, g, gate=E(()), sum_out=r, normed=r)),
        (ValueError, "both sides", bn(*[E(2, 3, 4, 8)] * 2, g, gate=E(2, 1, 4, 8), sum_out=E(2, 3, 4, 8), normed=E(2, 3, 4, 8))),
        (ValueError, "both sides", bn(*[E(2, 3, 4, 8)] * 2, g, gate=E(2, 1, 4, 1), sum_out=E(2, 3, 4, 8), normed=E(2, 3, 4, 8))),
        (ValueError, "more than one stride", bn(r, r, g, gate=E(2, 5, 8)[:, :3], sum_out=r, normed=r)),
        (ValueError, "contiguous last dim", bn(r, r, g, gate=E(2, 8, 3).transpose(1, 2), sum_out=r, normed=r)),
        (ValueError, "one GPU", bn(r, r, g, sum_out=r, normed=r)),
    ]:
        with pytest.raises(exc, match=match):
            fn()


def test_binding_refusals_without_the_extension_module(lib, monkeypatch):
    import mbrt
    from mbrt import _calls

    monkeypatch.setattr(mbrt, "_n", _calls)
    test_binding_refusals(lib)
