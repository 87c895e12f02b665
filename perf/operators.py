"""The transformer-layer operators of `mbrt`: the linear layer with its epilogue, the qkv split with
per-head norms and rotation, and attention through a sliding window with sinks.

Sizes are those of the model that the benchmark and the tests use (60 mel bands, 8 heads of 64, 384
features, feed-forward of 1536; an 8 s chunk has T = 801 frames and 48060 token rows), or generic:

  linear   act(x W^T + bias) + residual
  norm     qkv [B, N, (H + 2 Hkv) D] -> RMS-normed and rotated q and k, and v
  window   attention over the keys within a window of each query, and the first few keys
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _mbrt():
    path = str(Path(__file__).resolve().parent.parent / "mbr-cuda-tile_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mbrt

    return mbrt


def _linear(name, rows, k, n, dtype, act=None, bias=True, residual=False, out=None):
    return dict(name=name, kind="linear", rows=rows, k=k, n=n, dtype=dtype, out=out or dtype, act=act or "none",
                bias=bias, residual=residual)


def _norm(name, b, n, heads, kv_heads, d, dtype, pos0=0, order="bnhd"):
    return dict(name=name, kind="norm", b=b, n=n, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype, pos0=pos0,
                order=order)


def _window(name, b, nq, nk, heads, kv_heads, d, dtype, left, right, sinks, gate=False, ragged=False, start=-1,
            out=None):
    """left or right -1: no limit; start -1: the queries are the last of the keys."""
    return dict(name=name, kind="window", b=b, nq=nq, nk=nk, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype,
                left=left, right=right, sinks=sinks, gate=gate, ragged=ragged, start=start, out=out or dtype)


def listed():
    return [
        # the feed-forward entrance for one streamed frame: a row per band; latency
        _linear("linear_frame", 60, 384, 1536, "bf16", act="gelu"),
        # the fused qkv projection of an 8 s chunk
        _linear("linear_qkv", 48060, 384, 1536, "bf16", bias=False),
        # the feed-forward exit of that chunk, onto the residual stream
        _linear("linear_ff_out", 48060, 1536, 384, "bf16", residual=True),
        # its attention gates: one sigmoid per head and token
        _linear("linear_gate", 48060, 384, 8, "bf16", act="sigmoid"),
        # one band's projection into the model in full precision: a ragged number of columns
        _linear("linear_band", 801, 118, 384, "f32"),
        # one streamed frame of all bands, rotated at its place in the song
        _norm("norm_frame", 60, 1, 8, 8, 64, "bf16", pos0=1300),
        # the time attention's heads of an 8 s chunk
        _norm("norm_chunk", 60, 801, 8, 8, 64, "bf16"),
        # grouped key heads in full precision, an odd length, heads outside tokens
        _norm("norm_grouped", 7, 1301, 8, 2, 128, "f32", order="bhnd"),
        # the time attention of an 8 s chunk seen through half a second to each side, gated
        _window("window_chunk", 60, 801, 801, 8, 8, 64, "bf16", 50, 50, 8, gate=True),
        # one streamed frame against what each band has kept: lengths differ
        _window("window_stream", 60, 1, 1601, 8, 8, 64, "bf16", 800, 0, 4, ragged=True),
        # a whole song as one causal sequence with grouped heads
        _window("window_song", 2, 16389, 16389, 8, 2, 128, "f16", 1023, 0, 4),
        # one token against a long cache without a left limit
        _window("window_long", 1, 1, 200003, 8, 2, 64, "bf16", -1, 0, 0, out="f32"),
    ]


# ---- drawn cases ----------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "norm", "window"])
    if kind == "linear":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        k = rng.choice([384, 512, 1536, _log(rng, 16, 1536)])
        n = rng.choice([8, 384, 1536, _log(rng, 1, 1536)])
        top = 48060 * 1536 * 384 // (k * n * (8 if dtype == "f32" else 1))
        return dict(kind=kind, rows=_log(rng, 1, max(2, min(48060, top))), k=k, n=n, dtype=dtype,
                    out=rng.choice([dtype, dtype, "f32"]), act=rng.choice(["none", "none", "gelu", "sigmoid", "tanh"]),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.4)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    heads, kv_heads = rng.choice([(8, 8), (8, 8), (8, 2), (6, 3), (4, 1)])
    d = rng.choice([64, 64, 128, 32])
    if kind == "norm":
        dtype = rng.choice([dtype, "f32"])
        n = rng.choice([1, _log(rng, 1, 1601)])
        b = _log(rng, 1, max(2, min(60, 48060 * 64 // (n * d * (2 if dtype == "f32" else 1)))))
        return dict(kind=kind, b=b, n=n, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype,
                    pos0=rng.choice([0, rng.randint(0, 2000)]), order=rng.choice(["bnhd", "bhnd"]))
    sinks = rng.choice([0, 4, rng.randint(0, 80)])
    out = rng.choice([dtype, dtype, "f32"])
    form = rng.choice(["chunk", "stream", "long"])
    if form == "chunk":     # a chunk or a song through a window, causal or not
        n = _log(rng, 30, 4000)
        b = max(1, min(60, 30000 * 64 // (n * d)))
        left = _log(rng, 5, 700)
        right = rng.choice([0, left])
        return dict(kind="window", b=b, nq=n, nk=n, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype, left=left,
                    right=right, sinks=sinks, gate=rng.random() < 0.5, ragged=rng.random() < 0.3,
                    start=rng.choice([-1, 0]), out=out)
    nq = rng.choice([1, 1, 2, rng.randint(1, 16)])
    if form == "stream":    # a few frames against each band's cache
        nk = _log(rng, 20, 1601)
        return dict(kind="window", b=_log(rng, 1, 60 * 64 // d), nq=nq, nk=nk, heads=heads, kv_heads=kv_heads, d=d,
                    dtype=dtype, left=_log(rng, 16, 801), right=0, sinks=sinks, gate=rng.random() < 0.5,
                    ragged=rng.random() < 0.7, start=-1, out=out)
    nk = _log(rng, 2000, 100000)  # one token against a long cache
    return dict(kind="window", b=max(1, min(4, 100000 // nk)), nq=nq, nk=nk, heads=heads, kv_heads=min(kv_heads, 2),
                d=d, dtype=dtype, left=-1, right=0, sinks=0, gate=False, ragged=rng.random() < 0.5, start=-1, out=out)


# ---- inputs -----------------------------------------------------------------------------------

def _randn(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


def _lens(case, g):
    """Keys held per batch entry (int32), or None; at least as many as queries where those are the last."""
    if not case["ragged"]:
        return None
    lo = case["nk"] // 3 if case["start"] >= 0 else max(case["nq"], case["nk"] // 3)
    return torch.randint(lo, case["nk"] + 1, (case["b"],), generator=g, device=DEV, dtype=torch.int32)


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]
    if c["kind"] == "linear":
        return dict(x=_randn(g, (c["rows"], c["k"]), dt),
                    w=_randn(g, (c["n"], c["k"]), dt, std=1.0 / math.sqrt(c["k"])),
                    bias=_randn(g, (c["n"],), std=0.1) if c["bias"] else None,
                    residual=_randn(g, (c["rows"], c["n"]), DTYPES[c["out"]]) if c["residual"] else None)
    if c["kind"] == "norm":
        h = c["heads"] + 2 * c["kv_heads"]
        # cos and sin of position * frequency, the angle in 64 bits
        pos = torch.arange(c["pos0"] + c["n"], device=DEV, dtype=torch.float64)
        f = 10000.0 ** (-torch.arange(0, c["d"], 2, device=DEV, dtype=torch.float64) / c["d"])
        ang = pos[:, None] * f
        return dict(qkv=_randn(g, (c["b"], c["n"], h * c["d"]), dt),
                    q_gamma=_randn(g, (c["d"],), std=0.1, mean=1.0), k_gamma=_randn(g, (c["d"],), std=0.1, mean=1.0),
                    cos=torch.cos(ang).float(), sin=torch.sin(ang).float())
    # q, k of unit scale: scores of a trained model reach a few units, its maxima more
    return dict(q=_randn(g, (c["b"], c["nq"], c["heads"], c["d"]), dt, std=1.5),
                k=_randn(g, (c["b"], c["nk"], c["kv_heads"], c["d"]), dt),
                v=_randn(g, (c["b"], c["nk"], c["kv_heads"], c["d"]), dt), lens=_lens(c, g),
                gate=_randn(g, (c["b"], c["nq"], c["heads"]), dt) if c["gate"] else None)


def _head_views(case, order):
    """Buffers of the split's outputs, as [B, H, N, D] views of the given order."""
    c, dt = case, DTYPES[case["dtype"]]
    out = []
    for h in (c["heads"], c["kv_heads"], c["kv_heads"]):
        if order == "bhnd":
            out.append(torch.empty((c["b"], h, c["n"], c["d"]), dtype=dt, device=DEV))
        else:
            out.append(torch.empty((c["b"], c["n"], h, c["d"]), dtype=dt, device=DEV).permute(0, 2, 1, 3))
    return out


def prepare(case, seed):
    st = dict(case=case, **_inputs(case, seed))
    if own:
        m = _mbrt()
        st["mbrt"] = m
        odt = DTYPES[case["out"]] if "out" in case else None
        if case["kind"] == "linear":
            st["out"] = torch.empty((case["rows"], case["n"]), dtype=odt, device=DEV)
            st["act"] = {"none": m.ACT_NONE, "gelu": m.ACT_GELU_STD, "sigmoid": m.ACT_SIGMOID,
                         "tanh": m.ACT_TANH}[case["act"]]
        elif case["kind"] == "norm":
            st["heads_out"] = _head_views(case, case["order"])
        else:
            st["out"] = torch.empty((case["b"], case["nq"], case["heads"], case["d"]), dtype=odt, device=DEV)
            need = m.attention_window_workspace_bytes(case["b"], case["heads"], case["kv_heads"], case["nq"],
                                                      case["nk"], case["d"], _limit(case["left"]),
                                                      _limit(case["right"]), case["sinks"])
            st["workspace"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    return st


def _limit(x):
    return None if x < 0 else x


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    c = state["case"]
    kind = c["kind"]
    if own:
        m = state["mbrt"]
        if kind == "linear":
            return m.linear(state["x"], state["w"], state["bias"], state["out"], act=state["act"],
                            residual=state["residual"])
        if kind == "norm":
            q, k, v = state["heads_out"]
            m.split_qkv_norm_rotary(state["qkv"], state["q_gamma"], state["k_gamma"], state["cos"], state["sin"], q, k,
                                    v, c["heads"], kv_heads=c["kv_heads"], pos0=c["pos0"])
            return [q, k, v]
        return m.attention_window(state["q"], state["k"], state["v"], state["out"], left=_limit(c["left"]),
                                  right=_limit(c["right"]), sinks=c["sinks"], q_start=_limit(c["start"]),
                                  key_lens=state["lens"], gate=state["gate"], workspace=state["workspace"])
    if kind == "linear":
        return _plain_linear(state)
    if kind == "norm":
        return _plain_norm(state)
    return _plain_window(state)


def _plain_linear(s):
    c = s["case"]
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["act"] == "gelu":
        y = 0.5 * y * torch.erfc(y * -math.sqrt(0.5))
    elif c["act"] == "sigmoid":
        y = 1.0 / (1.0 + torch.exp(-y))
    elif c["act"] == "tanh":
        y = torch.tanh(y)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[c["out"]])


def _plain_norm(s):
    c = s["case"]
    b, n, h, kv, d = c["b"], c["n"], c["heads"], c["kv_heads"], c["d"]
    x = s["qkv"].float().view(b, n, h + 2 * kv, d)
    cos, sin = s["cos"][c["pos0"]:, None], s["sin"][c["pos0"]:, None]
    out = []
    for t, gamma in ((x[:, :, :h], s["q_gamma"]), (x[:, :, h:h + kv], s["k_gamma"])):
        t = t * (math.sqrt(d) * gamma) / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-12)
        x0, x1 = t[..., 0::2], t[..., 1::2]
        out.append(torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), dim=-1).flatten(-2))
    out.append(x[:, :, h + kv:])
    out = [t.to(s["qkv"].dtype).permute(0, 2, 1, 3) for t in out]
    return [t.contiguous() for t in out] if c["order"] == "bhnd" else out


def _starts(case, lens):
    """Position of each batch entry's first query, [B] int64 on the GPU."""
    if case["start"] >= 0:
        return torch.full((case["b"],), case["start"], device=DEV, dtype=torch.int64)
    if lens is None:
        return torch.full((case["b"],), case["nk"] - case["nq"], device=DEV, dtype=torch.int64)
    return lens.long() - case["nq"]


def _key_range(case, i0, i1):
    """First and last key that any query i0 .. i1-1 may see through its window, over all lengths."""
    c = case
    if c["start"] >= 0:
        first = last = c["start"]
    else:
        last = c["nk"] - c["nq"]
        first = max(0, c["nk"] // 3 - c["nq"]) if c["ragged"] else last
    lo = 0 if c["left"] < 0 else min(max(0, first + i0 - c["left"]), c["nk"])
    hi = c["nk"] - 1 if c["right"] < 0 else min(c["nk"] - 1, last + i1 - 1 + c["right"])
    return lo, hi


def _plain_window(s):
    c = s["case"]
    b, nq, nk, h, kv, d = c["b"], c["nq"], c["nk"], c["heads"], c["kv_heads"], c["d"]
    g = h // kv
    q = s["q"].float().view(b, nq, kv, g, d).permute(0, 2, 3, 1, 4)          # [B, KV, G, nq, D]
    k = s["k"].float().permute(0, 2, 3, 1).contiguous()                      # [B, KV, D, nk]
    v = s["v"].float().permute(0, 2, 1, 3).contiguous()                      # [B, KV, nk, D]
    start = _starts(c, s["lens"])
    length = torch.full((b,), nk, device=DEV, dtype=torch.int64) if s["lens"] is None else s["lens"].long()
    out = torch.empty((b, nq, h, d), dtype=DTYPES[c["out"]], device=DEV)
    step = 512
    for i0 in range(0, nq, step):
        i1 = min(nq, i0 + step)
        lo, hi = _key_range(c, i0, i1)
        sk = min(c["sinks"], lo, nk)
        keys = torch.cat((torch.arange(sk, device=DEV), torch.arange(lo, hi + 1, device=DEV)))
        kk, vv = (k, v) if keys.numel() == nk else (k[..., keys], v[:, :, keys])
        sc = (q[:, :, :, i0:i1].reshape(b, kv, g * (i1 - i0), d) @ kk).view(b, kv, g, i1 - i0, -1) / math.sqrt(d)
        p = start[:, None] + torch.arange(i0, i1, device=DEV)                # [B, rows]
        see = keys[None, None, :] < length[:, None, None]
        if c["right"] >= 0:
            see = see & (keys <= p[..., None] + c["right"])
        if c["left"] >= 0:
            see = see & ((keys >= p[..., None] - c["left"]) | (keys < c["sinks"]))
        sc = sc.masked_fill(~see[:, None, None], -math.inf)
        top = sc.amax(-1, keepdim=True).clamp_min(-3e38)
        e = torch.exp(sc - top)
        o = e.view(b, kv, g * (i1 - i0), -1) @ vv
        o = o.view(b, kv, g, i1 - i0, d) / e.sum(-1, keepdim=True).clamp_min(1e-38)
        o = o.permute(0, 3, 1, 2, 4).reshape(b, i1 - i0, h, d)
        if s["gate"] is not None:
            o = o / (1.0 + torch.exp(-s["gate"][:, i0:i1].float()))[..., None]
        out[:, i0:i1] = o
    return out


# ---- work and 64-bit results ---------------------------------------------------------------------

def _visible(case):
    """(query-key pairs, keys that some query sees), summed over the batch, full lengths assumed
    for ragged ones at their mean of two thirds."""
    c = case
    nk = c["nk"] if not c["ragged"] else (2 * c["nk"]) // 3
    start = c["start"] if c["start"] >= 0 else nk - c["nq"]
    pairs, seen = 0, 0
    for i in range(c["nq"]):
        p = start + i
        hi = nk - 1 if c["right"] < 0 else min(nk - 1, p + c["right"])
        lo = 0 if c["left"] < 0 else max(0, p - c["left"])
        n = max(0, hi - lo + 1) + max(0, min(c["sinks"], lo, hi + 1))
        pairs += n
        seen = max(seen, n) if i == 0 else min(nk, seen + 1)
    return pairs * c["b"], seen * c["b"]


def work(case):
    c = case
    if c["kind"] == "linear":
        m, k, n, es, os = c["rows"], c["k"], c["n"], SIZE[c["dtype"]], SIZE[c["out"]]
        return {"bytes": (m + n) * k * es + m * n * os * (2 if c["residual"] else 1) + 4 * n * c["bias"],
                "flops": 2 * m * n * k}
    if c["kind"] == "norm":
        e = c["b"] * c["n"] * (c["heads"] + 2 * c["kv_heads"]) * c["d"]
        return {"bytes": 2 * e * SIZE[c["dtype"]] + 4 * c["n"] * c["d"], "flops": 8 * e}
    pairs, seen = _visible(c)
    rows = c["b"] * c["nq"] * c["heads"]
    es = SIZE[c["dtype"]]
    return {"bytes": rows * c["d"] * (es + SIZE[c["out"]]) + 2 * seen * c["kv_heads"] * c["d"] * es,
            "flops": 4 * pairs * c["heads"] * c["d"]}


def exact(case, seed):
    """The definitions in 64 bits, on the GPU."""
    c, s = case, _inputs(case, seed)
    if c["kind"] == "linear":
        y = torch.empty((c["rows"], c["n"]), dtype=torch.float64, device=DEV)
        wt = s["w"].double().t().contiguous()
        for r0 in range(0, c["rows"], 8192):
            y[r0:r0 + 8192] = torch.mm(s["x"][r0:r0 + 8192].double(), wt)
        if c["bias"]:
            y += s["bias"].double()
        if c["act"] == "gelu":
            y = torch.special.ndtr(y) * y
        elif c["act"] == "sigmoid":
            y = torch.where(y < 0, torch.exp(y) / (1 + torch.exp(y)), 1 / (1 + torch.exp(-y)))
        elif c["act"] == "tanh":
            y = torch.tanh(y)
        return y + s["residual"].double() if c["residual"] else y
    if c["kind"] == "norm":
        h, kv, d = c["heads"], c["kv_heads"], c["d"]
        parts = s["qkv"].double().split([h * d, kv * d, kv * d], dim=-1)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[c["pos0"]:]
        out = []
        for t, gamma, hh in ((parts[0], s["q_gamma"], h), (parts[1], s["k_gamma"], kv), (parts[2], None, kv)):
            t = t.reshape(c["b"], c["n"], hh, d).transpose(1, 2)
            if gamma is not None:
                t = t * torch.rsqrt((t.square().sum(-1, keepdim=True) + 1e-12) / d) * gamma.double()
                z = torch.view_as_complex(t.reshape(*t.shape[:-1], d // 2, 2).contiguous()) * turn
                t = torch.view_as_real(z).flatten(-2)
            out.append(t)
        return out
    # attention, head by head and entry by entry over that entry's own keys
    b, nq, nk, h = c["b"], c["nq"], c["nk"], c["heads"]
    out = torch.zeros((b, nq, h, c["d"]), dtype=torch.float64, device=DEV)
    lens = [nk] * b if s["lens"] is None else s["lens"].tolist()
    step = 1024
    for e in range(b):
        kd, vd = s["k"][e].double().permute(1, 2, 0).contiguous(), s["v"][e].double().transpose(0, 1).contiguous()
        start = c["start"] if c["start"] >= 0 else lens[e] - nq
        for i0 in range(0, nq, step):
            i1 = min(nq, i0 + step)
            lo = 0 if c["left"] < 0 or c["sinks"] > 0 and start + i0 - c["left"] <= c["sinks"] \
                else min(max(0, start + i0 - c["left"]), lens[e])
            hi = lens[e] if c["right"] < 0 else max(min(lens[e], start + i1 + c["right"]), 0)
            cols = torch.arange(lo, hi, device=DEV)
            if lo > 0 and c["sinks"] > 0:
                cols = torch.cat((torch.arange(min(c["sinks"], lo), device=DEV), cols))
            if cols.numel() == 0:
                continue
            dist = cols - torch.arange(start + i0, start + i1, device=DEV)[:, None]
            hide = torch.zeros_like(dist, dtype=torch.bool)
            if c["right"] >= 0:
                hide |= dist > c["right"]
            if c["left"] >= 0:
                hide |= (dist < -c["left"]) & (cols >= c["sinks"])
            kc, vc = kd[:, :, cols].contiguous(), vd[:, cols].contiguous()
            for hd in range(h):
                kh = hd // (h // c["kv_heads"])
                z = torch.mm(s["q"][e, i0:i1, hd].double(), kc[kh]) * c["d"] ** -0.5
                z.masked_fill_(hide, -math.inf)
                out[e, i0:i1, hd] = torch.nan_to_num(torch.mm(torch.softmax(z, -1), vc[kh]), nan=0.0)
    if c["gate"]:
        out *= torch.sigmoid(s["gate"].double())[..., None]
    return out
