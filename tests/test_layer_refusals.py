"""CPU tests: what the transformer-layer entry points refuse, at the C-ABI and in the binding, before any launch.
Non-NULL pointers are stand-in addresses that are never read."""
from __future__ import annotations

import pytest

P = 0x10000
F32, F16, I64, BF16 = 0, 1, 2, 3
OK, ARG, DTYPE, SHAPE, ALIGN = 0, 1, 2, 3, 4


@pytest.fixture(scope="module")
def lib():
    import mbrt

    if not mbrt.LIB_PATH.exists():
        pytest.skip("libmbrt.so not built")
    return mbrt.lib()


def _err(lib):
    return lib.mbrt_last_error().decode()


def test_linear_arguments(lib):
    def call(x=P, dt=BF16, xs=64, w=P, ws=64, b=None, bdt=F32, r=None, rdt=F32, rs=0, out=P, odt=BF16, os=32, rows=10,
             k=64, n=32, act=0):
        return lib.mbrt_linear(x, dt, xs, w, ws, b, bdt, r, rdt, rs, out, odt, os, rows, k, n, act, None)

    assert call(dt=I64) == DTYPE and call(odt=I64) == DTYPE and call(b=P, bdt=I64) == DTYPE and call(r=P, rdt=4) == DTYPE
    assert call(act=5) == ARG and call(act=-1) == ARG and "activation" in _err(lib)
    assert call(rows=-1) == SHAPE and call(k=-1) == SHAPE and call(n=-1) == SHAPE
    assert call(k=1 << 28) == SHAPE and call(n=1 << 28, os=1 << 28) == SHAPE and call(rows=1 << 40) == SHAPE
    assert call(xs=-1) == SHAPE and call(ws=-8) == SHAPE and call(r=P, rs=-1) == SHAPE
    assert call(os=31) == SHAPE and "overlap" in _err(lib)
    assert call(x=None) == ARG and call(w=None) == ARG and call(out=None) == ARG
    assert call(x=P + 1) == ALIGN and call(w=P + 1) == ALIGN and call(out=P + 1) == ALIGN
    assert call(b=P + 2) == ALIGN and call(r=P + 1, rdt=BF16) == ALIGN
    assert call(rows=0) == OK and call(n=0) == OK  # nothing to do


def test_split_qkv_norm_rotary_arguments(lib):
    def call(qkv=P, dt=BF16, bs=1920, ns=192, qg=P, kg=P, gdt=F32, c=P, s=P, tdt=F32, n_pos=10, pos0=0, q=P, k=P, v=P,
             odt=BF16, st=(640, 64, 64, 640, 64, 64), B=1, N=10, H=1, KV=1, D=64):
        return lib.mbrt_split_qkv_norm_rotary(qkv, dt, bs, ns, qg, kg, gdt, c, s, tdt, n_pos, pos0, q, k, v, odt, *st, B, N, H,
                                              KV, D, 8.0, 1e-12, None)

    assert call(dt=I64) == DTYPE and call(odt=4) == DTYPE and call(gdt=F16) == DTYPE and call(tdt=F16) == DTYPE
    assert call(D=63) == SHAPE and call(D=0) == SHAPE and call(D=1 << 17) == SHAPE and "even" in _err(lib)
    assert call(B=-1) == SHAPE and call(N=-1) == SHAPE and call(H=0) == SHAPE and call(KV=0) == SHAPE
    for pos0, n_pos in ((1, 10), (-1, 10), (0, 9), (11, 10), (2 ** 62, 2 ** 62 + 5)):
        assert call(pos0=pos0, n_pos=n_pos) == SHAPE
        assert "positions" in _err(lib)
    assert call(st=(640, -64, 64, 640, 64, 64)) == SHAPE and call(ns=-1) == SHAPE
    assert call(st=(640, 64, 0, 640, 64, 64)) == SHAPE and "overlap" in _err(lib)
    assert call(st=(640, 64, 64, 640, 64, 0)) == SHAPE
    for name in ("qkv", "q", "k", "qg", "kg", "c", "s"):
        assert call(**{name: None}) == ARG
        assert call(**{name: P + 1}) == ALIGN
    assert call(v=P + 1) == ALIGN
    assert call(B=0) == OK and call(N=0) == OK


def test_attention_window_arguments(lib):
    def call(q=P, k=P, v=P, dt=BF16, B=1, H=4, KV=2, nq=100, nk=100, D=64, qs=(25600, 64, 256), ks=(12800, 64, 128), left=5,
             right=5, sinks=0, start=-1, lens=None, gate=None, gdt=F32, out=P, odt=BF16, os=(25600, 64, 256), scale=0.0,
             ws=None, wsb=0):
        return lib.mbrt_attention_window(q, k, v, dt, B, H, KV, nq, nk, D, *qs, *ks, left, right, sinks, start, lens, gate, gdt,
                                         1, out, odt, *os, scale, ws, wsb, None)

    assert call(dt=F32) == DTYPE and call(odt=I64) == DTYPE and call(gate=P, gdt=4) == DTYPE
    assert call(D=96) == SHAPE and "head_dim" in _err(lib)
    assert call(H=3) == SHAPE and call(KV=0) == SHAPE and call(H=0) == SHAPE and "key heads" in _err(lib)
    assert call(nq=-1) == SHAPE and call(nk=-1) == SHAPE and call(B=-1) == SHAPE and call(sinks=-1) == SHAPE
    assert call(nk=1 << 28) == SHAPE and call(nq=1 << 28) == SHAPE
    assert call(left=-2) == ARG and call(right=-2) == ARG and call(start=-2) == ARG and call(start=1 << 28) == ARG
    assert call(scale=-1.0) == ARG and call(scale=float("nan")) == ARG and call(scale=float("inf")) == ARG
    for name in ("q", "k", "v", "out"):
        assert call(**{name: None}) == ARG
        assert call(**{name: P + 8}) == ALIGN
    assert call(lens=P + 2) == ALIGN and call(gate=P + 2) == ALIGN
    assert call(qs=(25600, 64, 260)) == ALIGN and call(ks=(12800, 4, 128)) == ALIGN and call(os=(25600, 64, -256)) == ALIGN
    assert call(os=(25600, 0, 256)) == SHAPE and call(os=(25600, 64, 0)) == SHAPE and "overlap" in _err(lib)
    need = lib.mbrt_attention_window_workspace_bytes(1, 4, 2, 1, 50000, 64, -1, 0, 0)
    assert need > 0
    long = dict(nq=1, nk=50000, left=-1, right=0, qs=(256, 64, 256), os=(256, 64, 256))
    assert call(**long) == ARG and "workspace" in _err(lib)
    assert call(**long, ws=P, wsb=need - 1) == ARG and call(**long, ws=P + 2, wsb=need) == ARG
    assert call(B=0) == OK and call(nq=0) == OK


def test_workspace_bytes(lib):
    f = lib.mbrt_attention_window_workspace_bytes
    assert f(2, 4, 2, 500, 500, 64, 10, 10, 0) == 0     # many queries
    assert f(0, 4, 2, 1, 500, 64, 10, 10, 0) == 0 and f(1, 4, 2, 0, 500, 64, 10, 10, 0) == 0
    for bad in ((1, 4, 3, 1, 500, 64), (1, 4, 2, 1, 500, 60), (1, 4, 2, -1, 500, 64), (-1, 4, 2, 1, 5, 64)):
        assert f(*bad, 10, 10, 0) == -1
    # a share's rows: D sums, a maximum and a sum each
    assert f(1, 8, 2, 1, 100000, 64, -1, 0, 0) % (8 * 66 * 4) == 0
    # any window may be narrower than the keys are many: more than the keys need is never asked for
    assert f(1, 8, 2, 1, 100000, 64, 100, 0, 0) <= f(1, 8, 2, 1, 100000, 64, -1, 0, 0)


def test_binding_refusals(lib):
    import torch

    import mbrt

    x, w, out = torch.empty(6, 8), torch.empty(5, 8), torch.empty(6, 5)
    lin = lambda *a, **k: (lambda: mbrt.linear(*a, stream=0, **k))
    qkv, g, c = torch.empty(2, 3, 4 * 8), torch.empty(8), torch.empty(3, 4)
    q4, k4 = torch.empty(2, 2, 3, 8), torch.empty(2, 1, 3, 8)
    spl = lambda *a, **k: (lambda: mbrt.split_qkv_norm_rotary(*a, stream=0, **k))
    q, k = torch.empty(2, 3, 4, 64, dtype=torch.bfloat16), torch.empty(2, 7, 2, 64, dtype=torch.bfloat16)
    win = lambda *a, **kw: (lambda: mbrt.attention_window(*a, stream=0, **kw))
    ln = torch.zeros(2, dtype=torch.int32)
    for exc, match, fn in [
        (ValueError, r"\[N, K\]", lin(x, w[:, :7], out=out)),
        (ValueError, r"\[N, K\]", lin(x, w[0], out=out)),
        (ValueError, "differ in dtype", lin(x, w.half(), out=out)),
        (ValueError, r"residual \[\.\., N\]", lin(x, w, out=out[:5])),
        (ValueError, r"residual \[\.\., N\]", lin(x, w, out=out, residual=out[:, :4])),
        (ValueError, r"bias \[N\]", lin(x, w, torch.empty(4), out)),
        (ValueError, "contiguous last dim", lin(torch.empty(8, 6).t(), w, out=out)),
        (ValueError, "contiguous last dim", lin(x, w, out=torch.empty(5, 6).t())),
        (ValueError, "more than one stride", lin(torch.empty(4, 3, 8)[:, :2], w, out=torch.empty(4, 2, 5))),
        (ValueError, "disagree", lin(x, w, out=out, out_dtype=torch.half)),
        (TypeError, "torch.bool", lin(x.bool(), w.bool(), out=out)),
        (TypeError, "Tensor", lin(x, w, 1, out)),
        (ValueError, "one GPU", lin(x, w, out=out)),
        (ValueError, r"\(H \+ 2 H_kv\) D", spl(qkv, g, g, c, c, q4, k4, k4, 3, kv_heads=1)),
        (ValueError, r"\(H \+ 2 H_kv\) D", spl(qkv[0], g, g, c, c, q4, k4, k4, 2, kv_heads=1)),
        (ValueError, r"q \[B, H, N, D\]", spl(qkv, g, g, c, c, k4, k4, k4, 2, kv_heads=1)),
        (ValueError, "dtype", spl(qkv, g, g, c, c, q4, k4, k4.half(), 2, kv_heads=1)),
        (ValueError, "strided alike", spl(qkv, g, g, c, c, q4, k4, torch.empty(2, 1, 6, 8)[:, :, ::2], 2, kv_heads=1)),
        (ValueError, "gammas", spl(qkv, g[:7], g, c, c, q4, k4, k4, 2, kv_heads=1)),
        (ValueError, "cos, sin", spl(qkv, g, g, c, c[:2], q4, k4, k4, 2, kv_heads=1)),
        (ValueError, "contiguous last dim", spl(qkv, g, g, c, c, torch.empty(2, 2, 8, 3).transpose(2, 3), k4, k4, 2, kv_heads=1)),
        (ValueError, "one GPU", spl(qkv, g, g, c, c, q4, k4, k4, 2, kv_heads=1)),
        (ValueError, "expected q", win(q[0], k, k, q)),
        (ValueError, "expected q", win(q, k[:1], k[:1], q)),
        (ValueError, "dtype", win(q, k, k.half(), q)),
        (ValueError, "strided alike", win(q, k, torch.empty(2, 14, 2, 64, dtype=torch.bfloat16)[:, ::2], q)),
        (ValueError, "expected out", win(q, k, k, q[:, :2])),
        (ValueError, "key_lens", win(q, k, k, q, key_lens=ln.long())),
        (ValueError, "key_lens", win(q, k, k, q, key_lens=ln[:1])),
        (ValueError, "gate", win(q, k, k, q, gate=torch.empty(2, 3, 2))),
        (ValueError, "left", win(q, k, k, q, left=-1)),
        (ValueError, "q_start", win(q, k, k, q, q_start=-1)),
        (ValueError, "one GPU", win(q, k, k, q)),
    ]:
        with pytest.raises(exc, match=match):
            fn()
    with pytest.raises(ValueError):
        mbrt.attention_window_workspace_bytes(1, 4, 3, 1, 10, 64)


def test_binding_refusals_without_the_extension_module(lib, monkeypatch):
    import mbrt
    from mbrt import _calls

    monkeypatch.setattr(mbrt, "_n", _calls)
    test_binding_refusals(lib)


def test_linear_refuses_an_output_within_its_inputs(lib):
    far = [(k + 1) << 32 for k in range(4)]

    def call(x=far[0], w=far[1], b=None, r=None, out=far[2], xs=64, ws=64, rs=64, os=64, rows=100, dt=BF16, odt=BF16,
             rdt=BF16):
        return lib.mbrt_linear(x, dt, xs, w, ws, b, F32, r, rdt, rs, out, odt, os, rows, 64, 64, 0, None)

    def refused(**kw):
        return call(**kw) == ARG and "overlaps" in _err(lib)

    size = 2 * 100 * 64
    for at in (-size + 2, -2, 0, 2, size - 2):   # from one shared element at the front to one at the end
        assert refused(out=far[0] + at) and refused(r=far[3], out=far[3] + (at or 2))
    for at in (-size + 2, 0, 2 * 64 * 64 - 2):
        assert refused(out=far[1] + at)
    for at in (-size + 2, 0, 4 * 64 - 2):
        assert refused(b=far[3], out=far[3] + at)
    # the residual's place in another type or other rows
    assert refused(r=far[2], rdt=F16) and refused(r=far[2], rs=0) and refused(r=far[2], rs=128)
    # columns of one matrix of 128 of which x and out share one, or which meet at other strides; one row for all
    assert refused(xs=128, os=128, out=far[0] + 2 * 63) and refused(xs=128, os=128, out=far[0] - 2 * 63)
    assert refused(xs=100, os=128, out=far[0] + 2 * 64) and refused(xs=0, out=far[0] - 2 * 64 * 50)


def test_window_scale_beyond_float(lib):
    def call(scale):
        return lib.mbrt_attention_window(P, P, P, BF16, 1, 1, 1, 4, 4, 64, 256, 64, 64, 256, 64, 64, 5, 0, 0, -1, None, None, F32, 1,
                                         None, BF16, 256, 64, 64, scale, None, 0, None)

    assert call(3e38) == ARG and "scale" in _err(lib)      # in powers of 2 it is infinite
    assert call(2e38) == ARG and "NULL" in _err(lib)       # accepted: the next refusal is out's


def test_calls_too_large_for_one_launch(lib):
    """2^32 threads and more, which the hardware's launch cannot hold, are refused by size before the launch fails."""
    far = [(k + 1) << 48 for k in range(4)]
    for dt, rows, k, n in ((BF16, 1 << 32, 64, 64), (BF16, 1 << 33, 64, 8), (F32, 1 << 33, 64, 8), (F16, 1 << 32, 64, 1000)):
        assert lib.mbrt_linear(far[0], dt, 0, far[1], k, None, F32, None, F32, 0, far[2], dt, n, rows, k, n, 0, None) == SHAPE
        assert "too many" in _err(lib)
    for B, nq, nk in ((1 << 24, 1, 16), (1 << 20, 2000, 16)):
        assert lib.mbrt_attention_window(far[0], far[1], far[2], BF16, B, 1, 1, nq, nk, 64, nq * 64, 64, 64, 0, 0, 64, 5, 0, 0, -1,
                                         None, None, F32, 1, far[3], BF16, nq * 64, 64, 64, 0.0, None, 0, None) == SHAPE
        assert "too many" in _err(lib)
