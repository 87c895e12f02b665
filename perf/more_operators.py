"""The operators of `mbrt` for a transformer layer held in 4 bits: quantisation to microscaled 4-bit floats
(MXFP4 of the OCP Microscaling Formats specification v1.0), the linear layer of such weights, and the norms
before and after a block with its gate and residual scale.

Sizes are those of the model that the benchmark and the tests use (60 mel bands, 384 features, feed-forward of
1536; an 8 s chunk has T = 801 frames and 48060 token rows), or generic:

  norm      residual + alpha * layer_scale * gate * norm(update), and that sum's own norm
  quantize  rows to 4-bit codes with a scale per 32 features, and the values that those stand for
  product   act(x W^T + bias) + residual for W in 4 bits, x in 4 bits or not
  feed      norm into 4 bits, the feed-forward's two products with 4 bits between them
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "mx": 17 / 32}


def _mbrt():
    path = str(Path(__file__).resolve().parent.parent / "mbr-cuda-tile_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mbrt

    return mbrt


def _norm(name, b, n, d, stream, update, out, gate="none", post=True, scaled=False, alpha=1.0):
    """gate: none, token (one logit per row), batch (features of each batch entry), full."""
    return dict(name=name, kind="norm", b=b, n=n, d=d, stream=stream, update=update, out=out, gate=gate, post=post,
                scaled=scaled, alpha=alpha)


def _quantize(name, rows, k, dtype):
    return dict(name=name, kind="quantize", rows=rows, k=k, dtype=dtype)


def _product(name, rows, k, n, x, out="bf16", act="none", bias=True, residual=False):
    return dict(name=name, kind="product", rows=rows, k=k, n=n, x=x, out=out, act=act, bias=bias, residual=residual)


def _feed(name, b, n, d, ff, stream):
    return dict(name=name, kind="feed", b=b, n=n, d=d, ff=ff, stream=stream)


def listed():
    return [
        # one streamed frame of all bands behind the attention: latency
        _norm("norm_frame", 60, 1, 384, "bf16", "bf16", "bf16", gate="token"),
        # an 8 s chunk with its residual stream in full precision and a learned scale per feature
        _norm("norm_chunk", 60, 801, 384, "f32", "bf16", "bf16", scaled=True),
        # features gated per batch entry, as a conditioned block has them
        _norm("norm_batch", 4, 4003, 512, "f16", "f16", "f16", gate="batch", alpha=0.5),
        # an odd width with a gate of its own for every value
        _norm("norm_odd", 7, 1301, 1001, "f32", "f32", "f32", gate="full"),
        # the hidden activations of an 8 s chunk's feed-forward
        _quantize("quantize_hidden", 48060, 1536, "bf16"),
        # one band's ragged features in full precision
        _quantize("quantize_band", 801, 118, "f32"),
        # the feed-forward entrance for one streamed frame, weights alone in 4 bits: latency
        _product("product_frame", 60, 384, 1536, "bf16", act="gelu"),
        # one token through a large layer: the weights have to be read
        _product("product_token", 1, 4096, 16384, "bf16"),
        # the fused qkv projection of an 8 s chunk, activations in 4 bits
        _product("product_qkv", 48060, 384, 1536, "mx", bias=False),
        # a large square product onto the residual stream
        _product("product_square", 4096, 4096, 4096, "mx", residual=True),
        # the feed-forward of one streamed frame
        _feed("feed_frame", 60, 1, 384, 1536, "bf16"),
        # the feed-forward of an 8 s chunk
        _feed("feed_chunk", 60, 801, 384, 1536, "f32"),
    ]


# ---- drawn cases ----------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "product", "product", "feed"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "norm":
        d = rng.choice([384, 512, 1536, _log(rng, 16, 4096)])
        rows = _log(rng, 1, max(2, min(48060, 48060 * 384 // d)))
        b = min(rows, rng.choice([1, 4, 60, rng.randint(1, 60)]))
        stream = rng.choice([dtype, "f32"])
        return dict(kind=kind, b=b, n=max(1, rows // b), d=d, stream=stream, update=dtype,
                    out=rng.choice([dtype, dtype, "f32"]), gate=rng.choice(["none", "token", "batch", "full"]),
                    post=rng.random() < 0.7, scaled=rng.random() < 0.5, alpha=rng.choice([1.0, 0.5]))
    if kind == "quantize":
        k = rng.choice([384, 1536, _log(rng, 16, 8192)])
        return dict(kind=kind, rows=_log(rng, 1, max(2, min(48060, 48060 * 1536 // (2 * k)))), k=k, dtype=dtype)
    if kind == "product":
        x = rng.choice(["mx", "mx", dtype])
        k = rng.choice([384, 512, 1536, _log(rng, 16, 4096)])
        n = rng.choice([384, 1536, _log(rng, 1, 4096)])
        top = 48060 * 1536 * 384 // (k * n * (8 if x == "f32" else 1))
        return dict(kind=kind, rows=_log(rng, 1, max(2, min(48060, top))), k=k, n=n, x=x,
                    out=rng.choice(["bf16", "bf16", "f16", "f32"]), act=rng.choice(["none", "none", "gelu", "sigmoid"]),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.4)
    d = rng.choice([384, 512, _log(rng, 32, 1024)])
    ff = rng.choice([1536, 4 * d, _log(rng, 32, 4096)])
    rows = _log(rng, 1, max(2, min(48060, 48060 * 384 * 1536 // (d * ff))))
    b = min(rows, rng.choice([1, 4, 60]))
    return dict(kind=kind, b=b, n=max(1, rows // b), d=d, ff=ff, stream=rng.choice(["f32", "bf16"]))


# ---- inputs -----------------------------------------------------------------------------------

def _randn(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


def _features(g, shape, dtype):
    """Activations: some features are much larger than others."""
    spread = torch.exp(0.7 * torch.randn(shape[-1], generator=g, device=DEV))
    return (torch.randn(shape, generator=g, device=DEV) * spread).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = case
    if c["kind"] == "quantize":
        return dict(x=_features(g, (c["rows"], c["k"]), DTYPES[c["dtype"]]))
    if c["kind"] == "product":
        xt = torch.bfloat16 if c["x"] == "mx" else DTYPES[c["x"]]
        return dict(x=_features(g, (c["rows"], c["k"]), xt),
                    w=_randn(g, (c["n"], c["k"]), std=1.0 / math.sqrt(c["k"])),
                    bias=_randn(g, (c["n"],), std=0.1) if c["bias"] else None,
                    residual=_randn(g, (c["rows"], c["n"]), DTYPES[c["out"]]) if c["residual"] else None)
    b, n, d = c["b"], c["n"], c["d"]
    if c["kind"] == "feed":
        return dict(residual=_features(g, (b, n, d), DTYPES[c["stream"]]),
                    update=_randn(g, (b, n, d), torch.bfloat16),
                    post_gamma=_randn(g, (d,), std=0.1, mean=1.0), gamma=_randn(g, (d,), std=0.1, mean=1.0),
                    up=_randn(g, (c["ff"], d), std=1.0 / math.sqrt(d)), up_bias=_randn(g, (c["ff"],), std=0.1),
                    down=_randn(g, (d, c["ff"]), std=1.0 / math.sqrt(c["ff"])), down_bias=_randn(g, (d,), std=0.1))
    shape = {"token": (b, n, 1), "batch": (b, 1, d), "full": (b, n, d)}.get(c["gate"])
    return dict(residual=_features(g, (b, n, d), DTYPES[c["stream"]]),
                update=_randn(g, (b, n, d), DTYPES[c["update"]], std=0.7),
                post_gamma=_randn(g, (d,), std=0.1, mean=1.0) if c["post"] else None,
                gamma=_randn(g, (d,), std=0.1, mean=1.0),
                layer_scale=_randn(g, (d,), std=0.05, mean=0.3) if c["scaled"] else None,
                gate=_randn(g, shape, DTYPES[c["update"]]) if shape else None)


def prepare(case, seed):
    c, st = case, dict(case=case, **_inputs(case, seed))
    if own:
        m = st["mbrt"] = _mbrt()
        for name in ("w", "up", "down"):        # weights are quantised once
            if name in st:
                st[name] = m.mx_quantize(st[name])
        if c["kind"] == "product":
            if c["x"] == "mx":
                st["x"] = m.mx_quantize(st["x"])
            st["out"] = torch.empty((c["rows"], c["n"]), dtype=DTYPES[c["out"]], device=DEV)
            st["act"] = {"none": m.ACT_NONE, "gelu": m.ACT_GELU_STD, "sigmoid": m.ACT_SIGMOID}[c["act"]]
        elif c["kind"] == "quantize":
            st["held"] = m.mx_empty((c["rows"], c["k"]), device=DEV)
            st["out"] = torch.empty((c["rows"], c["k"]), dtype=DTYPES[c["dtype"]], device=DEV)
        else:
            st["sum"] = torch.empty_like(st["residual"])
            if c["kind"] == "norm":
                st["out"] = torch.empty((c["b"], c["n"], c["d"]), dtype=DTYPES[c["out"]], device=DEV)
            else:
                st["normed"] = m.mx_empty((c["b"], c["n"], c["d"]), device=DEV)
                st["hidden"] = m.mx_empty((c["b"], c["n"], c["ff"]), device=DEV)
                st["out"] = torch.empty((c["b"], c["n"], c["d"]), dtype=torch.bfloat16, device=DEV)
    else:
        for name in ("w", "up", "down"):
            if name in st:
                st[name] = _held(st[name])
        if c["kind"] == "product" and c["x"] == "mx":
            st["x"] = _held(st["x"])
    torch.cuda.synchronize()
    return st


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        m = s["mbrt"]
        if kind == "norm":
            return list(m.block_norm(s["residual"], s["update"], s["gamma"], post_gamma=s["post_gamma"], gate=s["gate"],
                                     gate_is_logit=c["gate"] == "token", layer_scale=s["layer_scale"], alpha=c["alpha"],
                                     sum_out=s["sum"], normed=s["out"]))
        if kind == "quantize":
            m.mx_quantize(s["x"], out=s["held"])
            return m.mx_dequantize(s["held"], out=s["out"])
        if kind == "product":
            return m.mx_linear(s["x"], s["w"], s["bias"], s["out"], act=s["act"], residual=s["residual"])
        m.block_norm(s["residual"], s["update"], s["gamma"], post_gamma=s["post_gamma"], sum_out=s["sum"],
                     normed=s["normed"])
        m.mx_linear(s["normed"], s["up"], s["up_bias"], s["hidden"], act=m.ACT_GELU_STD)
        m.mx_linear(s["hidden"], s["down"], s["down_bias"], s["out"])
        return [s["sum"], s["out"]]
    if kind == "norm":
        return [t.to(dt) for t, dt in zip(_plain_norm(s, c), (DTYPES[c["stream"]], DTYPES[c["out"]]))]
    if kind == "quantize":
        return _held(s["x"]).to(DTYPES[c["dtype"]])
    if kind == "product":
        return _plain_product(s["x"].float(), s["w"], s["bias"], c["act"], s["residual"]).to(DTYPES[c["out"]])
    h, normed = _plain_norm(s, dict(c, alpha=1.0, gate="none"))
    hidden = _held(_plain_product(_held(normed), s["up"], s["up_bias"], "gelu"))
    return [h.to(DTYPES[c["stream"]]), _plain_product(hidden, s["down"], s["down_bias"]).to(torch.bfloat16)]


def _held(x):
    """The f32 values that x [.., K] stands for in 4 bits."""
    k = x.shape[-1]
    t = x.double()
    if k % 32:
        t = torch.cat((t, t.new_zeros((*t.shape[:-1], 32 - k % 32))), -1)
    t = t.unflatten(-1, (-1, 32))
    # the power of two of the largest value, two below it so that it falls into [4, 8)
    e = torch.frexp(t.abs().amax(-1, keepdim=True)).exponent - 3
    e = torch.where(t.abs().amax(-1, keepdim=True) > 0, e, -127).clamp(-127, 127)
    one = torch.ones((), dtype=torch.float64, device=t.device)
    t = t * torch.ldexp(one, -e)
    a = t.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    t = torch.copysign((torch.round(a / step) * step).clamp_max(6.0), t) * torch.ldexp(one, e)
    return t.flatten(-2)[..., :k].float()


def _rms(t, gamma):
    return t * (math.sqrt(t.shape[-1]) * gamma) / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-12)


def _plain_norm(s, c):
    """The sum as it is stored, in f32, and its norm."""
    u = s["update"].float()
    if s["post_gamma"] is not None:
        u = _rms(u, s["post_gamma"])
    if s.get("layer_scale") is not None:
        u = u * s["layer_scale"]
    if s.get("gate") is not None:
        g = s["gate"].float()
        u = u * (1.0 / (1.0 + torch.exp(-g)) if c["gate"] == "token" else g)
    h = (s["residual"].float() + c["alpha"] * u).to(s["residual"].dtype).float()
    return h, _rms(h, s["gamma"])


def _plain_product(x, w, bias, act="none", residual=None):
    y = torch.matmul(x, w.t())
    if bias is not None:
        y = y + bias
    if act == "gelu":
        y = 0.5 * y * torch.erfc(y * -math.sqrt(0.5))
    elif act == "sigmoid":
        y = 1.0 / (1.0 + torch.exp(-y))
    return y if residual is None else y + residual.float()


# ---- work and 64-bit results ---------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "quantize":
        return {"bytes": 2 * c["rows"] * c["k"] * SIZE[c["dtype"]], "flops": 4 * c["rows"] * c["k"]}
    if c["kind"] == "product":
        m, k, n, os = c["rows"], c["k"], c["n"], SIZE[c["out"]]
        return {"bytes": int(m * k * SIZE[c["x"]] + n * k * SIZE["mx"]) + m * n * os * (2 if c["residual"] else 1),
                "flops": 2 * m * n * k}
    rows, d = c["b"] * c["n"], c["d"]
    if c["kind"] == "feed":
        return {"bytes": rows * d * (2 * SIZE[c["stream"]] + 2 + 2) + int(2 * d * c["ff"] * SIZE["mx"]),
                "flops": 4 * rows * d * c["ff"]}
    gate = {"none": 0, "token": rows, "batch": c["b"] * d, "full": rows * d}[c["gate"]]
    return {"bytes": rows * d * (2 * SIZE[c["stream"]] + SIZE[c["update"]] + SIZE[c["out"]]) + gate * SIZE[c["update"]],
            "flops": 10 * rows * d}


def _held64(x):
    """What x stands for in 4 bits, in 64 bits: every value's place among the eight magnitudes."""
    x = x.double()
    out = torch.empty_like(x)
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    for k0 in range(0, x.shape[-1], 32):
        t = x[..., k0:k0 + 32].contiguous()
        top = t.abs().max(dim=-1, keepdim=True).values
        exponent = (top.view(torch.int64) >> 52) - 1023 - 2          # floor(log2) - 2 of what is normal in 64 bits
        scale = torch.pow(2.0, exponent.clamp(-127, 127).double())
        a = t.abs() / scale
        # halfway values go to the even code
        place = ((a > 0.25).long() + (a >= 0.75).long() + (a > 1.25).long() + (a >= 1.75).long() + (a > 2.5).long()
                 + (a >= 3.5).long() + (a > 5).long())
        out[..., k0:k0 + 32] = torch.sign(t) * table[place] * scale
    return out


def _linear64(x, w, bias, act):
    y = torch.empty((x.shape[0], w.shape[0]), dtype=torch.float64, device=DEV)
    wt = w.t().contiguous()
    for r0 in range(0, x.shape[0], 8192):
        y[r0:r0 + 8192] = torch.mm(x[r0:r0 + 8192], wt)
    if bias is not None:
        y += bias.double()
    if act == "gelu":
        y = torch.special.ndtr(y) * y
    elif act == "sigmoid":
        y = torch.sigmoid(y)
    return y


def _norm64(x, gamma):
    return x * torch.rsqrt((x.square().sum(-1, keepdim=True) + 1e-12) / x.shape[-1]) * gamma.double()


def exact(case, seed):
    """The definitions in 64 bits, on the GPU."""
    c, s = case, _inputs(case, seed)
    if c["kind"] == "quantize":
        return _held64(s["x"])
    if c["kind"] == "product":
        x = _held64(s["x"]) if c["x"] == "mx" else s["x"].double()
        y = _linear64(x, _held64(s["w"]), s["bias"], c["act"])
        return y + s["residual"].double() if c["residual"] else y
    u = s["update"].double()
    if s["post_gamma"] is not None:
        u = _norm64(u, s["post_gamma"])
    if c["kind"] == "norm":
        if s["layer_scale"] is not None:
            u = s["layer_scale"].double() * u
        if s["gate"] is not None:
            g = s["gate"].double()
            u = (torch.sigmoid(g) if c["gate"] == "token" else g) * u
        u = c["alpha"] * u
    h = s["residual"].double() + u
    stored = h.to(s["residual"].dtype).double()      # the norm is of the sum as it is held
    normed = _norm64(stored, s["gamma"])
    if c["kind"] == "norm":
        return [h, normed]
    rows = c["b"] * c["n"]
    hidden = _held64(_linear64(_held64(normed.view(rows, -1)), _held64(s["up"]), s["up_bias"], "gelu"))
    y = _linear64(hidden, _held64(s["down"]), s["down_bias"], "none")
    return [h, y.view(c["b"], c["n"], c["d"])]
