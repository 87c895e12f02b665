"""Plain 64-bit forms of the transformer-layer operators on the CPU, with the bounds their 32-bit
evaluation has to keep.

Every bound is the sum of
 * f32 accumulation of n terms in any order: n U times the terms' magnitude, U = 2^-23 per operation (one step of f32,
   twice a correct rounding: the order inside a matrix instruction and its rounding are the hardware's);
 * what an approximated function adds, stated where it is used;
 * the one rounding of the output, finfo(dtype).eps / 2 of the value, and half the smallest subnormal of the type
   (fp16: 2^-25).
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -23


def half_step(dtype: torch.dtype, y: torch.Tensor) -> torch.Tensor:
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return y.abs() * (torch.finfo(dtype).eps / 2) + tiny


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} != {tuple(want.shape)}"
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN positions differ"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = ~(nan | inf)
    if not bool(ok.any()):
        return
    err, lim = (got - want).abs()[ok], bound.expand_as(want)[ok]
    worst = int(torch.argmax(err / lim))
    assert bool((err <= lim).all()), (f"{what}: off by {float(err[worst]):.3e}, bound {float(lim[worst]):.3e}, "
                                      f"value {float(want[ok][worst])!r}, {int((err > lim).sum())} of {err.numel()}")


def act64(y, act):
    """none, gelu_ref, gelu_std, sigmoid, tanh by their number, and a bound of their slope."""
    if act == 1:
        return 0.5 * y * torch.special.erfc(-y), 1.2   # max of 0.5 (1 + erf y) + y exp(-y^2) / sqrt(pi): 1.13
    if act == 2:
        return 0.5 * y * torch.special.erfc(-y * math.sqrt(0.5)), 1.2
    if act == 3:
        return torch.sigmoid(y), 0.25
    if act == 4:
        return torch.tanh(y), 1.0
    return y, 1.0


def linear(x, w, bias, act, residual, out_dtype):
    """(value, bound) of act(x w^T + bias) + residual."""
    xd, wd = x.detach().cpu().double(), w.detach().cpu().double()
    pre, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        pre, mag = pre + bias.cpu().double(), mag + bias.cpu().double().abs()
    y, slope = act64(pre, act)
    # K products and the bias
    bound = slope * (x.shape[-1] + 2) * U * mag
    # GELU: erf within 1.5e-7 (the 2-byte form, Abramowitz & Stegun 7.1.26, and f32 steps around it) or a few steps of
    # f32 times 0.5 |x|; sigmoid and tanh: exp of an f32 argument, |x| U relative and a few steps of values up to 1
    if act in (1, 2):
        bound = bound + 0.5 * pre.abs() * (1.5e-7 + 8 * U if out_dtype != torch.float32 else 8 * U)
    elif act in (3, 4):
        bound = bound + 8 * U + 0.3 * U * pre.abs().clamp_max(100)
    if residual is not None:
        y = y + residual.cpu().double()
        bound = bound + U * (y.abs() + residual.cpu().double().abs())
    return y, bound + half_step(out_dtype, y) + 1e-30


def qkv_norm(qkv, q_gamma, k_gamma, cos, sin, heads, kv_heads, scale, eps, pos0, out_dtype):
    """[(value, bound)] of q, k, v as [B, H, N, D]."""
    B, N, width = qkv.shape
    D = width // (heads + 2 * kv_heads)
    x = qkv.detach().cpu().double().view(B, N, heads + 2 * kv_heads, D)
    c, s = cos.cpu().double()[pos0:pos0 + N, None], sin.cpu().double()[pos0:pos0 + N, None]
    out = []
    for t, gamma in ((x[:, :, :heads], q_gamma), (x[:, :, heads:heads + kv_heads], k_gamma)):
        t = t * scale * gamma.cpu().double() / torch.sqrt((t * t).sum(-1, keepdim=True) + eps)
        x0, x1 = t[..., 0::2], t[..., 1::2]
        y = torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1).flatten(-2)
        # sum of squares: D terms, half of which reach its root; root, quotient, two products; the rotation's two
        # products and difference, of the pair's magnitude
        mag = torch.stack((x0.abs() * c.abs() + x1.abs() * s.abs(), x0.abs() * s.abs() + x1.abs() * c.abs()),
                          dim=-1).flatten(-2)
        bound = (D / 2 + 8) * U * mag + half_step(out_dtype, y) + 1e-30
        out.append((y.permute(0, 2, 1, 3), bound.permute(0, 2, 1, 3)))
    v = x[:, :, heads + kv_heads:].permute(0, 2, 1, 3)
    out.append((v, half_step(out_dtype, v)))
    return out


def visible(nq, nk, length, left, right, sinks, start):
    """[nq, nk] truth values of one batch entry."""
    p = (start if start is not None else length - nq) + torch.arange(nq)[:, None]
    j = torch.arange(nk)[None, :]
    see = (j < length) & (j >= 0)
    if right is not None:
        see = see & (j <= p + right)
    if left is not None:
        see = see & ((j >= p - left) | (j < sinks))
    return see.expand(nq, nk)


def window(q, k, v, out_dtype, left=None, right=None, sinks=0, q_start=None, key_lens=None, gate=None,
           gate_is_logit=True, scale=0.0):
    """(value, bound) as [B, N_q, H, D]; hidden keys and values are never touched."""
    B, nq, H, D = q.shape
    nk, KV = k.shape[1], k.shape[2]
    sc = scale if scale else 1.0 / math.sqrt(D)
    y, bound = torch.zeros((B, nq, H, D), dtype=torch.float64), torch.zeros((B, nq, H, D), dtype=torch.float64)
    qd, kd, vd = (t.detach().cpu().double() for t in (q, k, v))
    for b in range(B):
        length = nk if key_lens is None else min(max(int(key_lens[b]), 0), nk)
        see = visible(nq, nk, length, left, right, sinks, q_start)
        for i in range(nq):
            idx = torch.nonzero(see[i]).flatten()
            if idx.numel() == 0:
                continue
            kk = kd[b, idx].transpose(0, 1).repeat_interleave(H // KV, 0)   # [H, n, D]
            vv = vd[b, idx].transpose(0, 1).repeat_interleave(H // KV, 0)
            s = (kk @ qd[b, i, :, :, None]).squeeze(-1) * sc                # [H, n]
            mag = (kk.abs() @ qd[b, i, :, :, None].abs()).squeeze(-1) * sc
            e = torch.exp(s - s.amax(-1, keepdim=True))
            l = e.sum(-1, keepdim=True)
            y[b, i] = ((e / l)[:, None] @ vv).squeeze(1)
            spread = ((e / l)[:, None] @ vv.abs()).squeeze(1)
            # scores: D products and the scale, each score off by ds; weights off by 2 ds (score and maximum's), by
            # the two or three 2-byte values of the weights (2^-16 at most) and by exp2 and the sums (n + 16 steps)
            ds = (D + 4) * U * mag.amax(-1, keepdim=True) + 2 * U * s.abs().amax(-1, keepdim=True)
            bound[b, i] = (2 * ds + 2.0 ** -16 + (idx.numel() + 16) * U) * spread
    if gate is not None:
        g = torch.sigmoid(gate.cpu().double()) if gate_is_logit else gate.cpu().double()
        y = y * g[..., None]
        bound = bound * g.abs()[..., None] + y.abs() * (8 * U + 0.5 * U * (gate.cpu().double().abs()[..., None] if gate_is_logit else 0))
    return y, bound + half_step(out_dtype, y) + 1e-30


def gelu_by_formula(x, s):
    """x Phi by Abramowitz & Stegun 7.1.26 in 64 bits, erfc(z) = (a1 t + .. + a5 t^5) exp(-z^2), t = 1 / (1 + p z): the
    form that 2-byte results take, its own error included."""
    z = x.abs() * s
    t = 1.0 / (1.0 + 0.3275911 * z)
    p = t * (0.254829592 + t * (-0.284496736 + t * (1.421413741 + t * (-1.453152027 + t * 1.061405429))))
    return torch.where(x > 0, x, 0.0 * x) - 0.5 * x.abs() * p * torch.exp(-z * z)


def activation(x, act, out_dtype, short):
    """(value, bound) of an activation of f32 arguments, relative to the value far into the tails too, infinities and
    NaN included.  short: the forms that 2-byte results of 2-byte operands take."""
    x = x.detach().cpu().double()
    y, _ = act64(x, act)
    tiny = 2.0 ** -126 * (1 + x.abs().clamp_max(1e38))   # results below the normal numbers may be flushed
    if act in (1, 2):
        s = 1.0 if act == 1 else math.sqrt(0.5)
        z2 = (x * s).square().clamp_max(1e4)
        if short:
            # the formula's own error (at most 1.5e-7 |x| / 2), and f32: a dozen steps of erfc, three of z^2 through exp
            own = (gelu_by_formula(x, s) - y).abs()
            fine = torch.isfinite(x)
            assert bool((own[fine] <= 0.75e-7 * x.abs()[fine] + 1e-12).all())
            erfc = torch.special.erfc(x.abs() * s)
            bound = own + 0.5 * x.abs() * erfc * (16 + 4 * z2) * U + 2 * U * y.abs()
        else:
            # erfc within OpenCL's 16 steps; its argument's rounding, d ln erfc / d ln z < 2 z^2 + 1
            bound = y.abs() * (20 + 2 * (z2 + 1)) * U
    elif act == 3:
        bound = y.abs() * (8 + 3 * x.abs().clamp_max(200)) * U   # exp(-x): two roundings of its argument, rcp, add
    elif act == 4:
        # OpenCL's 5 steps of tanh; the short form's series (3.3e-7 at 1/4) and 1 - 2 / (exp + 1), which cancels to a quarter
        bound = y.abs() * (4e-7 + 16 * U if short else 8 * U)
    else:
        bound = 0.0 * y.abs()
    top = torch.finfo(out_dtype).max
    y = torch.where(y.abs() > top * (1 + torch.finfo(out_dtype).eps / 4), torch.copysign(torch.full_like(y, math.inf), y), y)
    return y, bound + half_step(out_dtype, y) + tiny
