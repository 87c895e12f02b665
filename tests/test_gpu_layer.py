"""GPU tests of the transformer-layer operators run together, as a model runs them: projection, head norms and
rotation, windowed attention with its gates, output projection onto the residual stream, norm and feed-forward."""
from __future__ import annotations

import math

import pytest
import torch

from gpu_util import say

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
H, DH, DIM, FF = 4, 64, 192, 512
WINDOW = dict(left=12, right=0, sinks=2)


def _weights(dtype):
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(s, generator=g)
    w = dict(qkv=r(3 * H * DH, DIM) / DIM ** 0.5, gate=r(H, DIM) / DIM ** 0.5, out=r(DIM, H * DH) / (H * DH) ** 0.5,
             up=r(FF, DIM) / DIM ** 0.5, down=r(DIM, FF) / FF ** 0.5)
    w = {k: v.to(dtype).cuda() for k, v in w.items()}
    w.update(gate_b=r(H).cuda(), up_b=(0.1 * r(FF)).cuda(), down_b=(0.1 * r(DIM)).cuda(), qg=(1 + 0.1 * r(DH)).cuda(),
             kg=(1 + 0.1 * r(DH)).cuda(), g1=(1 + 0.1 * r(DIM)).cuda(), g2=(1 + 0.1 * r(DIM)).cuda())
    return w


def _tables(n):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, DH, 2, dtype=torch.float64) / DH)
    return torch.cos(ang).float().cuda(), torch.sin(ang).float().cuda()


class Layer:
    """One layer over [B, n, DIM] frames that continue a cache of `cap` positions."""

    def __init__(self, B, cap, w):
        self.w, self.cos_sin, self.pos = w, _tables(cap), 0
        self.k, self.v = (torch.full((B, cap, H, DH), float("nan"), dtype=BF16, device="cuda") for _ in range(2))

    def __call__(self, x):
        import mbrt

        w, (B, n, _) = self.w, x.shape
        normed = torch.empty_like(x)
        mbrt.rms_norm(x, w["g1"], normed, math.sqrt(DIM))
        qkv, gate = mbrt.linear(normed, w["qkv"]), mbrt.linear(normed, w["gate"], w["gate_b"])
        at = slice(self.pos, self.pos + n)
        q = torch.empty((B, n, H, DH), dtype=BF16, device="cuda")
        mbrt.split_qkv_norm_rotary(qkv, w["qg"], w["kg"], *self.cos_sin, q.permute(0, 2, 1, 3),
                                   self.k[:, at].permute(0, 2, 1, 3), self.v[:, at].permute(0, 2, 1, 3), H, pos0=self.pos)
        o = mbrt.attention_window(q, self.k, self.v, q_start=self.pos, gate=gate, **WINDOW)
        mbrt.linear(o.view(B, n, H * DH), w["out"], out=x, residual=x)
        mbrt.rms_norm(x, w["g2"], normed, math.sqrt(DIM))
        hidden = mbrt.linear(normed, w["up"], w["up_b"], act=mbrt.ACT_GELU_STD)
        mbrt.linear(hidden, w["down"], w["down_b"], out=x, residual=x)
        self.pos += n
        return x


def _reference(x, w):
    """The layer in 64 bits, with every stored value rounded to bf16 as the calls store it."""
    r = lambda t: t.to(BF16).double()
    w = {k: v.cpu().double() for k, v in w.items()}
    x, (B, n, _) = x.cpu().double(), x.shape
    norm = lambda t, g: t * math.sqrt(t.shape[-1]) * g / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-12)
    cos, sin = (t.cpu().double()[:, None] for t in _tables(n))

    def turn(t):
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    y = r(norm(x, w["g1"]))
    qkv, gate = r(y @ w["qkv"].t()).view(B, n, 3, H, DH), r(y @ w["gate"].t() + w["gate_b"])
    q, k, v = r(turn(norm(qkv[:, :, 0], w["qg"]))), r(turn(norm(qkv[:, :, 1], w["kg"]))), qkv[:, :, 2]
    d = torch.arange(n)[None, :] - torch.arange(n)[:, None]
    see = (d <= 0) & ((d >= -WINDOW["left"]) | (torch.arange(n)[None, :] < WINDOW["sinks"]))
    s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) / math.sqrt(DH)
    o = torch.matmul(torch.softmax(s.masked_fill(~see, -math.inf), -1), v.transpose(1, 2)).transpose(1, 2)
    o = r(o * torch.sigmoid(gate)[..., None]).reshape(B, n, H * DH)
    x = r(o @ w["out"].t() + x)
    h = r(torch.nn.functional.gelu(r(norm(x, w["g2"])) @ w["up"].t() + w["up_b"]))
    return r(h @ w["down"].t() + w["down_b"] + x)


def _frames(B, n):
    return torch.randn((B, n, DIM), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()


# Both sides round at the same places; where a value falls next to a border the two round apart, one step of bf16
# (2^-7 relative), which reaches the output through products that average it out.  One stored value in every ten or so
# differs by a step at worst, so the output's own last step plus one in the residual's size bounds what is seen:
# 2^-7 of the value and 2^-6 of the output's RMS.
def _close(got, want):
    rms = float(want.square().mean().sqrt())
    err = (got.cpu().double() - want).abs()
    lim = 2.0 ** -7 * want.abs() + 2.0 ** -6 * rms
    assert bool((err <= lim).all()), float((err / lim).max())


@pytest.mark.parametrize("B,n", [(2, 70), (5, 33)])
def test_whole_sequence(dev, B, n):
    say(f"layer B={B} n={n}")
    w = _weights(BF16)
    x = _frames(B, n)
    want = _reference(x, w)
    _close(Layer(B, n, w)(x.clone()), want)


def test_streamed_frame_by_frame(dev):
    """Frames one at a time and in uneven groups give what the whole sequence gives."""
    B, n = 3, 40
    w = _weights(BF16)
    x = _frames(B, n)
    want = _reference(x, w)
    layer, got, at = Layer(B, n, w), [], 0
    for step in [1] * 15 + [7, 1, 3, 14]:
        got.append(layer(x[:, at:at + step].clone()))
        at += step
    assert at == n
    _close(torch.cat(got, 1), want)


def test_captured_layer(dev):
    B, n = 2, 50
    w = _weights(BF16)
    x = _frames(B, n)
    layer = Layer(B, n, w)
    want = layer(x.clone()).clone()
    layer.pos = 0
    buf = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(buf)
    for _ in range(3):
        buf.copy_(x)
        graph.replay()
        eager = Layer(B, n, w)(x.clone())
        torch.cuda.synchronize()
        assert torch.equal(buf, want) and torch.equal(eager, want)
