"""The calls of pyext/calls.cpp through ctypes, for a Python or torch that the extension module
was not built for (it is bound to one of each; libmbrt.so is not).  Same functions, arguments,
checks and errors; a call takes about 5 us more of host time.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _abi

_DT = {torch.float32: _abi.F32, torch.float16: _abi.F16, torch.int64: _abi.I64, torch.bfloat16: _abi.BF16,
       torch.int32: _abi.I32}


def _tensors(*ts):
    for t in ts:
        if not isinstance(t, torch.Tensor):
            raise TypeError("mbrt: expected a torch.Tensor")


def _contig(*ts):
    _tensors(*(t for t in ts if t is not None))
    for t in ts:
        if t is not None and not t.is_contiguous():
            raise ValueError("mbrt: expected a contiguous tensor")


def _dt(t, none=None):
    if t is None:
        return none
    try:
        return _DT[t.dtype]
    except KeyError as e:
        raise TypeError(f"mbrt: unsupported dtype {t.dtype}") from e


def _p(t):
    return C.c_void_p(0 if t is None else t.data_ptr())


def _s(stream):
    return C.c_void_p(torch.cuda.current_stream().cuda_stream if stream is None else stream)


def _float(x):
    return C.c_double(x).value  # a number as the C-ABI takes it: no text


def fill(t, value, stream):
    _tensors(t)
    _contig(t)
    _abi.call("mbrt_fill", _p(t), _dt(t), t.numel(), _float(value), _s(stream))


def strided_copy(src, dst, stream):
    _tensors(src, dst)
    _contig(dst)
    if src.shape != dst.shape:
        raise ValueError("strided_copy: shape mismatch")
    m = _abi.StridedMeta()
    m.ndim = src.dim()
    for d in range(src.dim()):
        m.dst_shape[d] = src.shape[d]
        m.src_strides[d] = src.stride(d)
    _abi.call("mbrt_strided_copy", _p(src), _p(dst), _dt(src), C.byref(m), _s(stream))


def pad(src, out, before, value, reflect, stream):
    _tensors(src, out)
    _contig(src, out)
    m = _abi.PadMeta()
    m.ndim = src.dim()
    for d in range(src.dim()):
        m.src_shape[d] = src.shape[d]
        m.dst_shape[d] = out.shape[d]
        m.pad_before[d] = before[d]
    if reflect:
        _abi.call("mbrt_pad_reflect", _p(src), _p(out), _dt(src), C.byref(m), _s(stream))
    else:
        _abi.call("mbrt_pad_const", _p(src), _p(out), _dt(src), C.byref(m), _float(value), _s(stream))


def cat(srcs, dim, out, stream):
    srcs = list(srcs)
    _tensors(out, *srcs)
    _contig(out, *srcs)
    dim = dim % out.dim()
    outer = inner = 1
    for d in range(dim):
        outer *= out.shape[d]
    for d in range(dim + 1, out.dim()):
        inner *= out.shape[d]
    arr = (_abi.CatSrc * len(srcs))()
    off = 0
    for i, s in enumerate(srcs):
        arr[i].ptr = s.data_ptr()
        arr[i].dim_size = s.shape[dim]
        arr[i].dim_offset = off
        off += s.shape[dim]
    _abi.call("mbrt_cat", _p(out), arr, len(srcs), outer, out.shape[dim], inner * out.element_size(), _s(stream))


def rms_norm(x, gamma, out, scale, eps, stream):
    _tensors(x, gamma, out)
    _contig(x, gamma, out)
    dim = x.shape[-1]
    _abi.call("mbrt_rms_norm", _p(x), _dt(x), _p(gamma), _dt(gamma), _p(out), _dt(out), x.numel() // dim, dim,
              _float(scale), _float(eps), _s(stream))


def residual_add_rms_norm(residual, update, gamma, sum_out, normed, scale, eps, stream):
    _tensors(residual, update, gamma, normed)
    _contig(residual, update, gamma, sum_out, normed)
    dim = residual.shape[-1]
    _abi.call("mbrt_residual_add_rms_norm", _p(residual), _p(update), _dt(residual), _p(gamma), _dt(gamma), _p(sum_out),
              _dt(sum_out, _dt(residual)), _p(normed), _dt(normed), residual.numel() // dim, dim, _float(scale),
              _float(eps), _s(stream))


def bias_act(x, bias, out, act, stream):
    _tensors(x, out)
    _contig(x, bias, out)
    cols = x.shape[-1]
    _abi.call("mbrt_bias_act", _p(x), _dt(x), _p(bias), _dt(bias, _abi.F32), _p(out), _dt(out), x.numel() // cols, cols,
              act, _s(stream))


def glu(x, out, stream):
    _tensors(x, out)
    _contig(x, out)
    full = x.shape[-1]
    if full % 2:
        raise ValueError("glu_last_dim: last dimension must be even")
    _abi.call("mbrt_glu_last_dim", _p(x), _dt(x), _p(out), _dt(out), x.numel() // full, full // 2, _s(stream))


def gate_merge(attn, gate, out, layout, gate_is_logit, stream):
    _tensors(attn, gate, out)
    _contig(attn, gate, out)
    if attn.dim() != 4:
        raise ValueError("gate_merge: expected a 4-d attention output")
    if layout == _abi.LAYOUT_BHND:
        B, H, N, D = attn.shape
    else:
        B, N, H, D = attn.shape
    _abi.call("mbrt_sigmoid_gate_merge", _p(attn), _dt(attn), _p(gate), _dt(gate), int(bool(gate_is_logit)), _p(out),
              _dt(out), B, H, N, D, layout, _s(stream))


def softmax(x, out, scale, stream):
    _tensors(x, out)
    _contig(x, out)
    cols = x.shape[-1]
    _abi.call("mbrt_softmax_rows", _p(x), _dt(x), _p(out), _dt(out), x.numel() // cols, cols, _float(scale), _s(stream))


def split_qkv_rotary(qkv, cos, sin, q, k, v, heads, stream):
    _tensors(qkv, cos, sin, q, k, v)
    _contig(qkv, cos, sin, q, k, v)
    if qkv.dim() != 3:
        raise ValueError("split_qkv_rotary: expected qkv [B, N, 3 H D]")
    B, N, three_hd = qkv.shape
    _abi.call("mbrt_split_qkv_heads_rotary", _p(qkv), _dt(qkv), _p(cos), _p(sin), _dt(cos), _p(q), _p(k), _p(v), _dt(q),
              B, N, heads, three_hd // (3 * heads), q.shape[2], _s(stream))


def attention_ex(q, k, v, sizes, strides, cos, sin, gate, gate_is_logit, out, scale, p_precision, stream):
    _tensors(q, k, v, out, *(t for t in (cos, sin, gate) if t is not None))
    _abi.call("mbrt_attention_ex", _p(q), _p(k), _p(v), _dt(q), *sizes, *strides, _p(cos), _p(sin), _dt(cos, _abi.F32),
              _p(gate), _dt(gate, _abi.F32), int(bool(gate_is_logit)), _p(out), _dt(out), _float(scale), p_precision,
              _s(stream))


def _gpu(*ts):
    """The device of these tensors, which a call is made on."""
    ts = [t for t in ts if t is not None]
    for t in ts:
        if t.device.type != "cuda" or t.device != ts[0].device:
            raise ValueError("mbrt: expected tensors on one GPU")
    return torch.cuda.device(ts[0].device)


def _unit_last(*ts):
    for t in ts:
        if t is not None and t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError("mbrt: expected a contiguous last dim")


def _alike(a, b):
    """Strides that are used, the same in both (those of a single index are not)."""
    return not a.numel() or all(x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n > 1)


def _row_stride(t, op="linear"):
    """The one stride between the rows of [.., n] (0 where there is one row)."""
    span, stride = 1, 0
    for d in range(t.dim() - 2, -1, -1):
        if t.shape[d] == 1:
            continue
        if t.numel() and span > 1 and t.stride(d) != span * stride:
            raise ValueError(f"{op}: the rows of a tensor lie at more than one stride")
        if span == 1:
            stride = t.stride(d)
        span *= t.shape[d]
    return stride


def linear(x, weight, bias, out, act, residual, stream):
    _tensors(x, weight, out, *(t for t in (bias, residual) if t is not None))
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError("linear: expected x [.., K] and weight [N, K]")
    N, K = weight.shape
    if x.dtype != weight.dtype:
        raise ValueError("linear: x and weight differ in dtype")
    want = x.shape[:-1] + (N,)
    if out.shape != want or residual is not None and residual.shape != want:
        raise ValueError("linear: expected out and residual [.., N]")
    if bias is not None and bias.shape != (N,):
        raise ValueError("linear: expected bias [N]")
    _unit_last(x, weight, out, residual, bias)
    rows = 1
    for s in x.shape[:-1]:
        rows *= s
    ws = weight.stride(0) if N > 1 else 0
    os = _row_stride(out) if rows > 1 else N
    args = (_p(x), _dt(x), _row_stride(x), _p(weight), ws, _p(bias), _dt(bias, _abi.F32), _p(residual),
            _dt(residual, _abi.F32), 0 if residual is None else _row_stride(residual), _p(out), _dt(out), os, rows, K, N,
            act)
    with _gpu(x, weight, bias, residual, out):
        _abi.call("mbrt_linear", *args, _s(stream))


def split_qkv_norm_rotary(qkv, q_gamma, k_gamma, cos, sin, q, k, v, heads, kv_heads, scale, eps, pos0, stream):
    _tensors(qkv, q_gamma, k_gamma, cos, sin, q, k, *(t for t in (v,) if t is not None))
    if qkv.dim() != 3 or heads < 1 or kv_heads < 1 or qkv.shape[2] % (heads + 2 * kv_heads):
        raise ValueError("split_qkv_norm_rotary: expected qkv [B, N, (H + 2 H_kv) D]")
    B, N, width = qkv.shape
    D = width // (heads + 2 * kv_heads)
    if q.shape != (B, heads, N, D) or k.shape != (B, kv_heads, N, D) or v is not None and v.shape != k.shape:
        raise ValueError("split_qkv_norm_rotary: expected q [B, H, N, D] and k, v [B, H_kv, N, D]")
    if q.dtype != k.dtype or v is not None and v.dtype != k.dtype:
        raise ValueError("split_qkv_norm_rotary: q, k and v differ in dtype")
    if v is not None and not _alike(k, v):
        raise ValueError("split_qkv_norm_rotary: k and v must be strided alike")
    if q_gamma.shape != (D,) or k_gamma.shape != (D,) or q_gamma.dtype != k_gamma.dtype:
        raise ValueError("split_qkv_norm_rotary: expected gammas [D] of one dtype")
    if cos.dim() != 2 or cos.shape[1] != D // 2 or sin.shape != cos.shape or sin.dtype != cos.dtype:
        raise ValueError("split_qkv_norm_rotary: expected cos, sin [n_pos, D/2] of one dtype")
    _contig(q_gamma, k_gamma, cos, sin)
    _unit_last(qkv, q, k, v)
    args = (_p(qkv), _dt(qkv), qkv.stride(0), qkv.stride(1), _p(q_gamma), _p(k_gamma), _dt(q_gamma), _p(cos), _p(sin),
            _dt(cos), cos.shape[0], pos0, _p(q), _p(k), _p(v), _dt(q), *q.stride()[:3], *k.stride()[:3], B, N, heads,
            kv_heads, D, _float(scale), _float(eps))
    with _gpu(qkv, q_gamma, k_gamma, cos, sin, q, k, v):
        _abi.call("mbrt_split_qkv_norm_rotary", *args, _s(stream))


def attention_window(q, k, v, out, left, right, sinks, q_start, key_lens, gate, gate_is_logit, scale, workspace,
                     stream):
    _tensors(q, k, v, out, *(t for t in (key_lens, gate, workspace) if t is not None))
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("attention_window: expected q [B, N_q, H, D] and k, v [B, N_k, H_kv, D]")
    B, nq, H, D = q.shape
    nk, KV = k.shape[1], k.shape[2]
    if k.shape != (B, nk, KV, D) or v.shape != k.shape:
        raise ValueError("attention_window: expected q [B, N_q, H, D] and k, v [B, N_k, H_kv, D]")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("attention_window: q, k and v differ in dtype")
    if not _alike(k, v):
        raise ValueError("attention_window: k and v must be strided alike")
    if out.shape != q.shape:
        raise ValueError("attention_window: expected out [B, N_q, H, D]")
    if key_lens is not None and (key_lens.shape != (B,) or key_lens.dtype != torch.int32):
        raise ValueError("attention_window: expected key_lens [B] int32")
    if gate is not None and gate.shape != (B, nq, H):
        raise ValueError("attention_window: expected gate [B, N_q, H]")
    _unit_last(q, k, v, out)
    _contig(key_lens, gate, workspace)
    qs, ks, os = q.stride(), k.stride(), out.stride()
    args = (_p(q), _p(k), _p(v), _dt(q), B, H, KV, nq, nk, D, qs[0], qs[2], qs[1], ks[0], ks[2], ks[1], left, right,
            sinks, q_start, _p(key_lens), _p(gate), _dt(gate, _abi.F32), int(bool(gate_is_logit)), _p(out), _dt(out),
            os[0], os[2], os[1], _float(scale), _p(workspace),
            0 if workspace is None else workspace.numel() * workspace.element_size())
    with _gpu(q, k, v, out, key_lens, gate, workspace):
        _abi.call("mbrt_attention_window", *args, _s(stream))


def _mx(op, codes, scales, lead, features):
    """Row strides of codes and scales that hold [*lead, features] in 4 bits."""
    blocks = -(-features // 32)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError("mbrt: expected codes and scales of dtype torch.uint8")
    if codes.shape != (*lead, 16 * blocks) or scales.shape != (*lead, blocks):
        raise ValueError(f"{op}: expected codes [.., 16 ceil(n / 32)] and scales [.., ceil(n / 32)]")
    _unit_last(codes, scales)
    return _row_stride(codes, op), _row_stride(scales, op)


def _rows(lead):
    n = 1
    for s in lead:
        n *= s
    return n


def mx_quantize(x, codes, scales, features, stream):
    _tensors(x, codes, scales)
    if x.dim() < 1 or x.shape[-1] != features:
        raise ValueError("mx_quantize: expected x [.., n]")
    cs, ss = _mx("mx_quantize", codes, scales, x.shape[:-1], features)
    _unit_last(x)
    args = (_p(x), _dt(x), _row_stride(x, "mx_quantize"), _p(codes), cs, _p(scales), ss, _rows(x.shape[:-1]), features)
    with _gpu(x, codes, scales):
        _abi.call("mbrt_mx_quantize", *args, _s(stream))


def mx_dequantize(codes, scales, features, out, stream):
    _tensors(codes, scales, out)
    if out.dim() < 1 or out.shape[-1] != features:
        raise ValueError("mx_dequantize: expected out [.., n]")
    cs, ss = _mx("mx_dequantize", codes, scales, out.shape[:-1], features)
    _unit_last(out)
    args = (_p(codes), cs, _p(scales), ss, _p(out), _dt(out), _row_stride(out, "mx_dequantize"), _rows(out.shape[:-1]), features)
    with _gpu(codes, scales, out):
        _abi.call("mbrt_mx_dequantize", *args, _s(stream))


def mx_linear(x, x_scales, w, w_scales, K, bias, out, out_scales, act, residual, stream):
    _tensors(x, w, w_scales, out, *(t for t in (x_scales, bias, out_scales, residual) if t is not None))
    op = "mx_linear"
    if x.dim() < 1 or w.dim() != 2 or x_scales is None and x.shape[-1] != K:
        raise ValueError("mx_linear: expected x [.., K] and weight [N, K]")
    N, lead = w.shape[0], x.shape[:-1]
    ws, wss = _mx(op, w, w_scales, (N,), K)
    xs, xss = (_row_stride(x, op), 0) if x_scales is None else _mx(op, x, x_scales, lead, K)
    if out_scales is None and out.shape != (*lead, N) or residual is not None and residual.shape != (*lead, N):
        raise ValueError("mx_linear: expected out and residual [.., N]")
    os, oss = (_row_stride(out, op), 0) if out_scales is None else _mx(op, out, out_scales, lead, N)
    if bias is not None and bias.shape != (N,):
        raise ValueError("mx_linear: expected bias [N]")
    _unit_last(x, out, residual, bias)
    xdt = _dt(x) if x_scales is None else _abi.MXFP4
    odt = _dt(out) if out_scales is None else _abi.MXFP4
    args = (_p(x), xdt, xs, _p(x_scales), xss, _p(w), ws, _p(w_scales), wss, _p(bias), _dt(bias, _abi.F32), _p(residual),
            _dt(residual, _abi.F32), 0 if residual is None else _row_stride(residual, op), _p(out), odt, os, _p(out_scales), oss,
            _rows(lead), K, N, act)
    with _gpu(x, x_scales, w, w_scales, bias, residual, out, out_scales):
        _abi.call("mbrt_mx_linear", *args, _s(stream))


def _gate_rows(gate, like):
    """(columns, row stride, inner, period): row r of `like` [.., D] has the gate's row (r / inner) % period."""
    if gate is None:
        return 1, 0, 1, 1
    D = like.shape[-1]
    if not 1 <= gate.dim() <= like.dim() or gate.shape[-1] not in (1, D):
        raise ValueError("block_norm: expected gate [.., D] or [.., 1]")
    stride, inner, period, closed = 0, 1, 1, False
    for d in range(2, like.dim() + 1):
        n, m = like.shape[-d], gate.shape[-d] if d <= gate.dim() else 1
        if m not in (1, n):
            raise ValueError("block_norm: expected gate [.., D] or [.., 1]")
        if n == 1:
            continue
        if m == 1:
            if period == 1:
                inner *= n
            else:
                closed = True
            continue
        if closed:
            raise ValueError("block_norm: the gate's rows are shared on both sides of a dim that they do not share")
        if period > 1 and like.numel() and gate.stride(-d) != period * stride:
            raise ValueError("block_norm: the rows of a tensor lie at more than one stride")
        if period == 1:
            stride = gate.stride(-d)
        period *= n
    return gate.shape[-1], stride, max(inner, 1), max(period, 1)


def block_norm(residual, update, post_gamma, gate, gate_is_logit, layer_scale, gamma, sum_out, normed, normed_scales, alpha,
               post_scale, scale, eps, stream):
    _tensors(residual, update, *(t for t in (post_gamma, gate, layer_scale, gamma, sum_out, normed, normed_scales) if t is not None))
    op = "block_norm"
    if residual.dim() < 1 or residual.shape[-1] < 1 or update.shape != residual.shape or \
            sum_out is not None and sum_out.shape != residual.shape or \
            normed is not None and normed_scales is None and normed.shape != residual.shape:
        raise ValueError("block_norm: expected update, sum_out and normed [.., D]")
    lead, D = residual.shape[:-1], residual.shape[-1]
    if sum_out is not None and sum_out.dtype != residual.dtype:
        raise ValueError("block_norm: sum_out and residual differ in dtype")
    for t in (post_gamma, layer_scale, gamma):
        if t is not None and t.shape != (D,):
            raise ValueError("block_norm: expected gammas and layer_scale [D]")
    _contig(post_gamma, layer_scale, gamma)
    _unit_last(residual, update, sum_out, normed, gate)
    os, oss = (0, 0) if normed is None else (_row_stride(normed, op), 0) if normed_scales is None else \
        _mx(op, normed, normed_scales, lead, D)
    odt = _abi.MXFP4 if normed_scales is not None else _dt(normed, _abi.F32)
    cols, gs, inner, period = _gate_rows(gate, residual)
    f = _abi.F32
    args = (_p(residual), _dt(residual), _row_stride(residual, op), _p(update), _dt(update), _row_stride(update, op),
            _p(post_gamma), _dt(post_gamma, f), _p(gate), _dt(gate, f), cols, gs, inner, period, int(bool(gate_is_logit)),
            _p(layer_scale), _dt(layer_scale, f), _p(gamma), _dt(gamma, f), _p(sum_out),
            0 if sum_out is None else _row_stride(sum_out, op), _p(normed), odt, os, _p(normed_scales), oss, _rows(lead), D,
            _float(alpha), _float(post_scale), _float(scale), _float(eps))
    with _gpu(residual, update, post_gamma, gate, layer_scale, gamma, sum_out, normed, normed_scales):
        _abi.call("mbrt_block_norm", *args, _s(stream))


def stft(x, window, hop, center, normalized, out, n_fft, win_length, stream):
    _tensors(x, window, out)
    _contig(x, window, out)
    _abi.call("mbrt_stft", _p(x), _p(window), _p(out), x.shape[0], x.shape[1], n_fft, hop, win_length, window.numel(),
              int(bool(center)), int(bool(normalized)), _s(stream))


def istft(spec, window, hop, center, normalized, length, out, workspace, n_fft, win_length, stream):
    _tensors(spec, window, out, workspace)
    _contig(spec, window, out)
    if spec.dim() != 4:
        raise ValueError("istft: expected a spectrum [B, F, T, 2]")
    B, F, T, _ = spec.shape
    _abi.call("mbrt_istft", _p(spec), _dt(spec), _p(window), _p(out), B, F, T, n_fft, hop, win_length, window.numel(),
              int(bool(center)), int(bool(normalized)), length, _p(workspace),
              workspace.numel() * workspace.element_size(), _s(stream))


def chunk_accumulate(dest, weight_sum, src, window, offset, stream):
    _tensors(dest, weight_sum, src, window)
    _contig(dest, weight_sum, src, window)
    n = src.shape[-1]
    _abi.call("mbrt_chunk_accumulate", _p(dest), _p(weight_sum), _p(src), _p(window), src.numel() // max(n, 1), n,
              dest.shape[-1], offset, _s(stream))
