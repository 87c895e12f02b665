"""Microscaled 4-bit floats, their products and the norms around a block in plain 64-bit form on the CPU, with the bounds
that 32-bit evaluation has to keep (terms as in layer_ref.py)."""
from __future__ import annotations

import math

import torch

import layer_ref as ref

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
U = ref.U


def pad32(x):
    n = x.shape[-1]
    return torch.cat((x, x.new_zeros((*x.shape[:-1], -n % 32))), -1)


def scale_codes(top):
    """Of blocks with these largest magnitudes (64 bits)."""
    e = torch.frexp(top).exponent.long() - 1            # floor(log2)
    code = torch.where(top > 0, e - 2, -127).clamp(-127, 127) + 127
    return torch.where(torch.isfinite(top), code, 255)


def places(a):
    """Index into VALUES of magnitudes a, nearest, halfway ones to the even index, all past 5 to the last."""
    return ((a > 0.25).long() + (a >= 0.75).long() + (a > 1.25).long() + (a >= 1.75).long() + (a > 2.5).long()
            + (a >= 3.5).long() + (a > 5).long())


def quantize(x):
    """(codes [.., 32 ceil(n / 32)] one per feature, scale codes) of x [.., n]."""
    t = pad32(x.detach().cpu().double()).unflatten(-1, (-1, 32))
    top = t.abs().amax(-1)
    sc = scale_codes(torch.where(torch.isnan(t).any(-1), math.nan, top))
    a = torch.nan_to_num(t) * torch.ldexp(torch.ones((), dtype=torch.float64), 127 - sc)[..., None]
    return (places(a.abs()) + 8 * torch.signbit(t).long()).flatten(-2), sc


def unpack(codes):
    """One code per feature from bytes."""
    c = codes.detach().cpu().long()
    return torch.stack((c & 15, c >> 4), -1).flatten(-2)


def values(codes, scales, n):
    """What codes (one per feature) and scales stand for."""
    c = codes.cpu()
    v = VALUES[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    s = torch.ldexp(torch.ones((), dtype=torch.float64), scales.cpu().long() - 127)
    s = torch.where(scales.cpu() == 255, math.nan, s)
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)[..., :n]


def held(x):
    """The values that an MxTensor stands for, in 64 bits."""
    return values(unpack(x.codes), x.scales.detach().cpu().long(), x.features)


def check_held(got, want, bound, what=""):
    """An MxTensor against results known within a bound: every scale is that of a largest value within it, every code the
    nearest to a value within it, under that scale."""
    codes, sc, n = unpack(got.codes), got.scales.detach().cpu().long(), got.features
    w, b = pad32(want).unflatten(-1, (-1, 32)), pad32(bound.expand_as(want)).unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(w).all(-1)
    assert torch.equal(sc == 255, bad), f"{what}: NaN blocks differ"
    w, b = torch.nan_to_num(w), torch.nan_to_num(b)
    lo, hi = scale_codes((w.abs() - b).clamp_min(0).amax(-1)), scale_codes((w.abs() + b).amax(-1))
    ok = ((sc >= lo) & (sc <= hi)) | bad
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} scales differ"
    one = torch.ones((), dtype=torch.float64)
    inv, s = torch.ldexp(one, 127 - sc)[..., None], torch.ldexp(one, sc - 127)[..., None]
    q = lambda t: torch.sign(t) * VALUES[places(t.abs() * inv)] * s
    v = values(codes, torch.where(bad, 0, sc), codes.shape[-1]).unflatten(-1, (-1, 32))
    ok = ((v >= q(w - b)) & (v <= q(w + b))) | bad[..., None]
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} values are not the nearest"
    assert bool((codes[..., n:] & 7 == 0).all() | bad.any()), f"{what}: the last block is not filled with zeros"


# log2 Phi(-s t), s 1 or sqrt 2: rising powers of t, each an f32
TAIL = {2: [-0.999987721, -1.15126169, -0.458557367, -0.0537483469, 0.00834418833, -0.000874139543, 5.28514029e-05, -1.33747221e-06],
        1: [-0.999987721, -1.62812996, -0.917114735, -0.152023286, 0.0333767533, -0.00494488003, 0.000422811223, -1.51317709e-05]}


def gelu_by_tail(x, act):
    """(value, bound) of the form that results in 4 bits take, max(x, 0) - |x| 2^p(|x|), in 64 bits, and of its f32 evaluation."""
    t = x.abs()
    terms = [float(torch.tensor(c, dtype=torch.float32)) * t ** k for k, c in enumerate(TAIL[act])]
    p, mag = sum(terms), sum(v.abs() for v in terms)
    part = t * torch.exp2(p)
    # p: seven sums, each off by half a step of what the terms add up to at most; exp2 by two steps of its value, and 0 or one
    # step of 2^-149 where that is below 2^-126; the last sum
    dp = torch.nan_to_num(7 * mag * U, nan=0.0, posinf=0.0)
    return x.clamp(min=0) - part, part * (dp * math.log(2) * 1.01 + 4 * U) + t * 2.0 ** -126 + 2 * U * t


def linear(x, w, bias, act, residual, out_dtype):
    """(value, bound) for x, w tensors of values in 64 bits; out_dtype None: results in 4 bits, before their rounding."""
    y, bound = ref.linear(x, w, bias, act, residual, out_dtype or torch.bfloat16)
    if out_dtype is None:
        bound = bound - ref.half_step(torch.bfloat16, y)
        if act in (1, 2):   # a form of its own, off by at most 1.1e-7
            pre = x.detach().cpu().double() @ w.detach().cpu().double().t() + (0 if bias is None else bias.cpu().double())
            v, b = gelu_by_tail(pre, act)
            own = (v - ref.act64(pre, act)[0]).abs()
            assert bool((own <= 1.1e-7).all())
            bound = bound + own + b
        return y, bound
    # past the type's largest value by half a step and more: infinite
    top = torch.finfo(out_dtype).max * (1 + torch.finfo(out_dtype).eps / 4)
    return torch.where(y.abs() > top, torch.copysign(torch.full_like(y, math.inf), y), y), bound


def block_sum(residual, update, post_gamma, gate, gate_is_logit, layer_scale, alpha, post_scale, eps):
    """(value, bound) of the sum before its rounding."""
    u = update.detach().cpu().double()
    D = u.shape[-1]
    steps = 6.0
    if post_gamma is not None:
        # sum of squares: D terms, half of which reach its root; root and products
        u = u * post_scale * post_gamma.cpu().double() / torch.sqrt((u * u).sum(-1, keepdim=True) + eps)
        steps += D / 2 + 6
    if layer_scale is not None:
        u = u * layer_scale.cpu().double()
    if gate is not None:
        g = gate.detach().cpu().double()
        if gate_is_logit:   # exp of an f32 argument, a sum and a reciprocal
            steps = steps + 8 + 0.5 * g.abs()
            g = torch.sigmoid(g)
        u = u * g
    u = u * alpha
    h = residual.detach().cpu().double() + u
    return h, U * (steps * u.abs() + h.abs()) + 1e-38


def norm(h, gamma, scale, eps):
    h = h.detach().cpu().double()
    y = h * scale * gamma.cpu().double() / torch.sqrt((h * h).sum(-1, keepdim=True) + eps)
    return y, (h.shape[-1] / 2 + 8) * U * y.abs() + 1e-38
