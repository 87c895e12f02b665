"""GPU tests of the windowed attention against its 64-bit form over the visible keys alone."""
from __future__ import annotations

import math

import pytest
import torch

import layer_ref as ref
from gpu_util import say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(seed, shape, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def _qkv(seed, B, nq, nk, H, KV, D, dtype, std=1.5):
    return (_rand(seed, (B, nq, H, D), dtype, std), _rand(seed + 1, (B, nk, KV, D), dtype),
            _rand(seed + 2, (B, nk, KV, D), dtype))


def _case(B, nq, nk, H=2, KV=2, D=64, dtype=BF16, out_dtype=None, lens=None, gate=None, seed=0, **kw):
    import mbrt

    say(f"window B={B} nq={nq} nk={nk} H={H}/{KV} D={D} {dtype} out={out_dtype} lens={lens} gate={gate} {kw}")
    q, k, v = _qkv(seed, B, nq, nk, H, KV, D, dtype)
    kl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    gt = None if gate is None else _rand(9, (B, nq, H), gate)
    got = mbrt.attention_window(q, k, v, key_lens=kl, gate=gt, out_dtype=out_dtype, **kw)
    torch.cuda.synchronize()
    want, bound = ref.window(q, k, v, got.dtype, key_lens=kl, gate=gt, **kw)
    ref.check(got, want, bound, "window")
    return got


WINDOWS = [dict(left=0, right=0), dict(left=5, right=0), dict(left=5, right=5, sinks=3), dict(left=40, right=7, sinks=70),
           dict(right=0), dict(left=33), dict(), dict(left=200, right=0, sinks=4), dict(left=1000000, right=1000000)]


@pytest.mark.parametrize("kw", WINDOWS)
@pytest.mark.parametrize("n", [1, 2, 31, 64, 65, 150, 301])
def test_self_attention(dev, n, kw):
    _case(2, n, n, **kw)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KV", [(4, 4), (4, 1), (6, 2)])
def test_heads_and_types(dev, H, KV, D, dtype):
    _case(2, 100, 100, H, KV, D, dtype, left=20, right=0, sinks=2)
    _case(1, 100, 100, H, KV, D, dtype, F32, left=20, right=9)
    _case(2, 1, 90, H, KV, D, dtype, left=70, right=0, sinks=2)
    _case(2, 3, 90, H, KV, D, dtype, F32, right=0)


@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("gate", [None, F32, BF16, F16])
def test_gate_and_output_types(dev, out, gate):
    _case(2, 70, 70, 4, 2, 64, BF16, out, gate=gate, left=16, right=16)
    _case(2, 1, 70, 4, 2, 64, BF16, out, gate=gate, left=16, right=0)
    if gate is not None:
        _case(1, 5, 40, 4, 2, 64, BF16, out, gate=gate, gate_is_logit=False, left=16, right=0)


@pytest.mark.parametrize("nq", [1, 2, 7, 16, 17, 64])
@pytest.mark.parametrize("kw", [dict(left=300, right=0, sinks=4), dict(right=0), dict(left=40, right=3)])
def test_few_queries_against_a_cache(dev, nq, kw):
    _case(3, nq, 700, 4, 2, 64, BF16, lens=[700, 333, nq], **kw)
    _case(1, nq, 1300, 2, 1, 128, F16, **kw)


@pytest.mark.parametrize("nk", [255, 256, 257, 1025, 2049, 5000])
def test_shared_out_over_the_keys(dev, nk):
    """One token against caches that are divided among workgroups and joined."""
    import mbrt

    assert nk < 1024 or mbrt.attention_window_workspace_bytes(1, 2, 1, 1, nk, 64, None, 0) > 0
    _case(1, 1, nk, 2, 1, 64, BF16, F32, right=0)
    _case(1, 3, nk, 8, 1, 32, F16, right=0, left=nk - 100, sinks=5)
    _case(3, 1, nk, 4, 2, 128, BF16, F32, lens=[nk, nk // 3, 0], right=0)


@pytest.mark.parametrize("nq", [1, 40, 130])
def test_positions(dev, nq):
    """Queries before, among and behind the keys; rows that see nothing are zero."""
    for start in (0, 5, 100, 180, 400):
        got = _case(2, nq, 200, q_start=start, left=30, right=2)
        if start == 400:
            assert bool((got == 0).all())
    _case(1, nq, 200, q_start=300, left=30, right=0, sinks=3)   # the sinks alone
    _case(2, nq, 200, lens=[0, 3], left=10, right=0)            # fewer keys than queries, or none
    _case(2, nq, 200, lens=[0, 3], q_start=0)
    _case(2, nq, 200, lens=[-5, 10 ** 9])                       # lengths out of range are clamped


def test_no_keys_and_no_queries(dev):
    import mbrt

    q = _rand(1, (2, 5, 2, 64), BF16)
    none = torch.empty((2, 0, 2, 64), dtype=BF16, device="cuda")
    assert bool((mbrt.attention_window(q, none, none) == 0).all())
    assert mbrt.attention_window(q[:, :0], q, q).shape == (2, 0, 2, 64)
    assert mbrt.attention_window(q[:0], q[:0], q[:0]).shape == (0, 5, 2, 64)


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), 3e38])
@pytest.mark.parametrize("nq", [1, 90])
def test_what_is_hidden_may_hold_anything(dev, nq, fill):
    """Keys and values behind each length, before the window, and between the sinks and the window."""
    import mbrt

    B, nk, H = 2, 200, 2
    q, k, v = _qkv(1, B, nq, nk, H, H, 64, BF16)
    lens = torch.tensor([nk - 60, nk - 1], dtype=torch.int32, device="cuda")
    kw = dict(left=20, right=0, sinks=2)
    clean = mbrt.attention_window(q, k, v, key_lens=lens, **kw)
    for b in range(B):
        first = int(lens[b]) - nq - 20
        for t in (k, v):
            t[b, int(lens[b]):] = fill
            t[b, 2:max(2, first)] = fill
    got = mbrt.attention_window(q, k, v, key_lens=lens, **kw)
    assert torch.equal(got, clean)


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
def test_hidden_from_some_rows_only(dev, fill):
    """A value or key that one row of a tile sees and its neighbours do not: only the rows that see it change."""
    import mbrt

    n, H = 100, 2
    for nq in (n, 4):
        for which in ("k", "v"):
            q, k, v = _qkv(4, 1, nq, n, H, H, 64, BF16)
            clean = mbrt.attention_window(q, k, v, left=10, right=0)
            at = n - 2
            (k if which == "k" else v)[0, at, 0, 5] = fill
            got = mbrt.attention_window(q, k, v, left=10, right=0)
            sees = torch.arange(n - nq, n, device="cuda") >= at
            assert torch.equal(got[0, ~sees], clean[0, ~sees]) or \
                bool(((got[0, ~sees].double() - clean[0, ~sees].double()).abs() <= 2.0 ** -7).all())
            assert bool(torch.isfinite(got[0, ~sees]).all())
            assert torch.equal(got[0, :, 1], clean[0, :, 1])
            want, bound = ref.window(q, k, v, BF16, left=10, right=0)
            finite = torch.isfinite(want).all(-1)
            assert bool((torch.isfinite(got.cpu()).all(-1) == finite).all())
            got_f = torch.where(finite[..., None], got.cpu().double(), 0.0)
            ref.check(got_f, torch.where(finite[..., None], want, 0.0), torch.where(finite[..., None], bound, 1.0), which)


def test_everything_nan_ends_early(dev):
    """Rows that see NaN at once are NaN without a walk over their keys: 64 million query-key pairs here."""
    import mbrt

    q, k, v = _qkv(2, 1, 8000, 8000, 1, 1, 64, BF16)
    for t in (q, k, v):
        kept = t.clone()
        t.fill_(float("nan"))
        got = mbrt.attention_window(q, k, v, right=0)
        torch.cuda.synchronize()
        assert bool(torch.isnan(got).all())
        t.copy_(kept)


@pytest.mark.parametrize("nq", [1, 30])
def test_one_column_of_a_value_is_nan(dev, nq):
    """The other columns, and rows that do not see it, keep their values."""
    import mbrt

    for D in (32, 128):
        q, k, v = _qkv(8, 1, nq, 80, 2, 2, D, F16)
        v[0, 70, 1, 3] = float("nan")
        got = mbrt.attention_window(q, k, v, left=40, right=0).cpu()
        want, bound = ref.window(q, k, v, F16, left=40, right=0)
        ref.check(got, want, bound, "one column")


def test_large_scores_and_values(dev):
    """Scores far apart, values near the type's largest: the running maximum and sum must carry them."""
    import mbrt

    for dtype, big in ((BF16, 2e38), (F16, 6e4)):
        q, k, v = _qkv(3, 1, 70, 200, 2, 2, 64, dtype, std=20.0)
        v = (v.float().sign() * big).to(dtype)
        got = mbrt.attention_window(q, k, v, left=60, right=0, out_dtype=F32)
        want, bound = ref.window(q, k, v, F32, left=60, right=0)
        ref.check(got, want, bound, "large")


def test_views_of_a_projection_and_of_padded_outputs(dev):
    import mbrt

    B, n, H, D = 2, 120, 4, 64
    qkv = _rand(1, (B, n, 3, H, D), BF16)
    q, k, v = qkv.unbind(2)
    room = torch.full((B, n + 9, H, D), 7.0, dtype=BF16, device="cuda")
    for nq in (n, 2):
        room.fill_(7.0)
        out = room[:, 4:4 + nq]
        got = mbrt.attention_window(q[:, n - nq:], k, v, out, left=30, right=30, sinks=1)
        assert got is out
        want, bound = ref.window(q[:, n - nq:], k, v, BF16, left=30, right=30, sinks=1)
        ref.check(out, want, bound, "views")
        assert bool((room[:, :4] == 7).all() and (room[:, 4 + nq:] == 7).all())
    heads_first = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]
    want, bound = ref.window(q, k, v, BF16, left=30, right=0)
    ref.check(mbrt.attention_window(*heads_first, left=30, right=0), want, bound, "heads first")


def test_scale(dev):
    _case(1, 50, 50, left=9, right=0, scale=0.4)
    _case(1, 1, 50, left=9, right=0, scale=0.01)


def test_agrees_with_the_full_attention(dev):
    """No limits: the same as attention_bnhd, gate and all, within both sides' bounds."""
    import mbrt

    q, k, v = _qkv(1, 2, 130, 170, 4, 4, 64, BF16)
    gate = _rand(5, (2, 130, 4), F32)
    got = mbrt.attention_window(q, k, v, gate=gate, out_dtype=F32)
    full = mbrt.attention_bnhd(q, k, v, gate=gate, out_dtype=F32)
    _, bound = ref.window(q, k, v, F32, gate=gate)
    assert bool(((got.cpu().double().view(2, 130, 256) - full.cpu().double()).abs() <= 2 * bound.view(2, 130, 256)).all())


def test_a_long_cache_past_32_bits(dev):
    """Key rows whose offsets pass 2^32 bytes and 2^31 elements."""
    import mbrt

    nk, stride = 70016, 32768
    big = torch.empty(2 * nk * stride, dtype=BF16, device="cuda")
    k = big.as_strided((1, nk, 1, 64), (nk * stride, stride, 64, 1))
    v = big.as_strided((1, nk, 1, 64), (nk * stride, stride, 64, 1), nk * stride)
    k.copy_(_rand(1, (1, nk, 1, 64), BF16))
    v.copy_(_rand(2, (1, nk, 1, 64), BF16))
    for nq in (1, 100):
        q = _rand(3, (1, nq, 2, 64), BF16, 1.5)
        got = mbrt.attention_window(q, k, v, left=150, right=0, sinks=3)
        kc, vc = (torch.cat((t[:, :3], t[:, nk - nq - 150:]), 1).contiguous() for t in (k, v))
        want, bound = ref.window(q, kc, vc, BF16, left=150, right=0, sinks=3)
        ref.check(got, want, bound, "far keys")


def test_same_result_every_time_captured_and_on_other_streams(dev):
    """Two calls at once with workspaces of their own, and a captured one, against the plain call."""
    import mbrt

    q, k, v = _qkv(1, 1, 2, 6000, 4, 2, 64, BF16)
    qs, ks, vs = _qkv(2, 2, 200, 200, 4, 2, 64, BF16)
    want, wants = mbrt.attention_window(q, k, v, right=0), mbrt.attention_window(qs, ks, vs, left=30, right=0)
    need = mbrt.attention_window_workspace_bytes(1, 4, 2, 2, 6000, 64, None, 0)
    assert need > 0
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [mbrt.attention_window(q, k, v, right=0, stream=s) for s in streams for _ in range(3)]
    torch.cuda.synchronize()
    for t in got:
        assert torch.equal(t, want)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out, outs = torch.empty_like(want), torch.empty_like(wants)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mbrt.attention_window(q, k, v, out, right=0, workspace=ws)
        mbrt.attention_window(qs, ks, vs, outs, left=30, right=0)
    for _ in range(4):
        out.zero_(), outs.zero_()
        graph.replay()
        eager = mbrt.attention_window(q, k, v, right=0)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(outs, wants) and torch.equal(eager, want)


def test_scores_of_minus_infinity(dev):
    """A query that sees keys, none of which scores above -infinity, is NaN, as the softmax is; zeros are for those that
    see no key.  Where another key's score is finite the infinite ones have no weight."""
    inf = float("inf")
    import mbrt

    for dtype in (BF16, F16):
        for nq, nk in ((1, 90), (90, 90), (7, 90), (1, 5000), (2, 5000)):
            say(f"scores of -inf nq={nq} nk={nk} {dtype}")
            q, k, v = _qkv(5, 1, nq, nk, 2, 1, 64, dtype)
            q[..., 0] = 1
            k[:, nk - 1, 0, 0] = -inf
            # each query sees its own key alone, the last one an infinite one
            got = mbrt.attention_window(q, k, v, left=0, right=0).cpu()
            want = v[:, nk - nq:].expand(1, nq, 2, 64).clone().cpu()
            want[:, nq - 1] = float("nan")
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(got[:, :nq - 1], want[:, :nq - 1])
            # all keys but one
            k[..., 0] = -inf
            assert bool(torch.isnan(mbrt.attention_window(q, k, v)).all())
            k[:, 3, 0, 0] = 0.5
            got = mbrt.attention_window(q, k, v).cpu()
            assert torch.equal(got, v[:, 3:4].expand(1, nq, 2, 64).cpu())
            # queries behind every key: none is seen
            assert bool((mbrt.attention_window(q, k, v, q_start=nk + 50, left=9) == 0).all())
    q, k, v = _qkv(6, 1, 3, 200, 2, 2, 32, BF16)
    k[..., 0] = -inf
    q[..., 0] = 1
    gate = torch.ones((1, 3, 2), device="cuda")
    lens = torch.tensor([0], dtype=torch.int32, device="cuda")
    assert bool(torch.isnan(mbrt.attention_window(q, k, v, gate=gate)).all())
    assert bool((mbrt.attention_window(q, k, v, gate=gate, key_lens=lens) == 0).all())


def _sink_case(B, nq, nk, D, dtype, gap, seed):
    """Keys whose first scores `gap` above the others, which lie within half a unit, and whose first value is zero."""
    g = torch.Generator().manual_seed(seed)
    q = torch.zeros((B, nq, 2, D))
    q[..., 0] = math.sqrt(D)
    k = torch.zeros((B, nk, 2, D))
    k[..., 0] = torch.rand((B, nk, 2), generator=g) - 0.5
    k[:, 0, :, 0] = gap
    v = 0.5 + torch.rand((B, nk, 2, D), generator=g)
    v[:, 0] = 0
    return q.to(dtype).cuda(), k.to(dtype).cuda(), v.to(dtype).cuda()


@pytest.mark.parametrize("out", [F16, F32])
@pytest.mark.parametrize("gap", [8.0, 12.0, 14.0, 16.0, 18.0])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_weights_far_below_a_sink(dev, D, gap, out):
    """f16 heads whose output is made by weights far below the largest one: a sink of value zero."""
    import mbrt

    for B, nq, nk in ((1, 100, 1000), (1, 1, 1000), (1, 1, 20000), (128, 130, 600)):
        say(f"sink D={D} gap={gap} B={B} nq={nq} nk={nk} {out}")
        q, k, v = _sink_case(B, nq, nk, D, F16, gap, nk)
        got = mbrt.attention_window(q, k, v, out_dtype=out)
        s = k.cpu().double()[..., 0] * (float(q[0, 0, 0, 0]) / math.sqrt(D))   # [B, nk, 2]
        e = torch.exp(s - s.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
        vd = v.cpu().double()
        y = (p[..., None] * vd).sum(1)
        # scores: exact products but for the scale and exp2's argument, a few steps of `gap` each; the weights' two f16
        # values: 2^-22 of each weight, and half the smallest f16 number beside a largest one of 2^10 or more, 2^-35 of the
        # row's largest weight; sums: n steps
        spread, lost = y.abs(), p.amax(1)[..., None] * vd.abs().sum(1)
        bound = spread * (2.0 ** -22 + (6 * (gap + 1) + nk + 16) * ref.U) + 2.0 ** -35 * lost
        y, bound = (t[:, None].expand(B, nq, 2, D) for t in (y, bound))
        ref.check(got, y, bound + ref.half_step(out, y) + 1e-30, f"gap {gap}")


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F32)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_weights_add_up_to_one(dev, D, dtype, out):
    """Values that are all 1 give 1: what is lost of each weight shows, whatever the scores' rounding."""
    import mbrt

    for B, nq, nk in ((4, 300, 300), (8, 1, 5), (8, 16, 7)):
        say(f"weights D={D} {dtype} B={B} nq={nq} nk={nk}")
        q, k, _ = _qkv(7, B, nq, nk, 2, 2, D, dtype)
        v = torch.ones_like(k)
        got = mbrt.attention_window(q, k, v, left=2, right=0, out_dtype=out).cpu().double()
        # at most 3 weights, held to 2^-23 (f16 pairs; bf16 triples 2^-24); the same weights are summed in f32 on both sides:
        # 2 additions each, the product's order, the quotient and the products with it.  Queries before the first key: 0.
        want = (torch.arange(nk - nq, nk) >= 0).double()[None, :, None, None]
        assert float((got - want).abs().max()) <= 2.0 ** -23 + 8 * ref.U


@pytest.mark.parametrize("D", [32, 64, 128])
def test_weights_of_bf16_behind_a_border(dev, D):
    """2-byte outputs of values that are all 1, moved by their gate to just beside the border between 1 and 1 + 2^-7:
    they fall on the gate's side of it if the weights add up to 1 within what is moved."""
    import mbrt

    # queries against caches: three parts, 2^-24, and f32's sums as in the test above; tiles: two parts, 2^-17
    for B, nq, nk, off in ((64, 8, 40, 2.0 ** -24 + 10 * ref.U), (64, 1, 40, 2.0 ** -24 + 10 * ref.U),
                           (8, 300, 300, 2.0 ** -17 + 10 * ref.U)):
        say(f"border D={D} B={B} nq={nq} nk={nk}")
        q, k, _ = _qkv(11, B, nq, nk, 4, 2, D, BF16)
        v = torch.ones_like(k)
        for side, want in ((1 + off, 1 + 2.0 ** -7), (1 - off, 1.0)):
            gate = torch.full((B, nq, 4), (1 + 2.0 ** -8) * side, device="cuda")
            got = mbrt.attention_window(q, k, v, left=2, right=0, gate=gate, gate_is_logit=False)
            assert int((got != want).sum()) == 0


def _single_index_strides(t, dims):
    """The same view with strides of `dims`, of one index each, that nothing uses."""
    st = list(t.stride())
    for d in dims:
        assert t.shape[d] == 1
        st[d] = 8 * t.numel() + 3
    return t.as_strided(t.shape, st)


@pytest.mark.parametrize("path", ["native", "ctypes"])
def test_strides_that_nothing_uses(dev, path, monkeypatch):
    """Strides of dimensions of size 1 may be anything, and differ between keys and values."""
    import mbrt
    from mbrt import _calls

    if path == "ctypes":
        monkeypatch.setattr(mbrt, "_n", _calls)
    for B, nq, nk, H, KV, odd in ((1, 40, 60, 2, 2, (0,)), (3, 1, 60, 2, 1, (2,)), (1, 1, 1, 1, 1, (0, 1, 2)),
                                  (2, 1, 60, 4, 4, ())):
        say(f"single indices B={B} nq={nq} nk={nk} {H}/{KV}")
        q, k, v = _qkv(3, B, nq, nk, H, KV, 64, BF16)
        want = mbrt.attention_window(q, k, v, left=30, right=0)
        qd = [d for d in range(3) if q.shape[d] == 1]
        out = _single_index_strides(torch.empty_like(want), qd)
        got = mbrt.attention_window(_single_index_strides(q, qd), k, _single_index_strides(v, odd), out, left=30, right=0)
        assert torch.equal(got, want)


@pytest.mark.parametrize("nq,nk,H,KV", [(65, 3000, 8, 2), (257, 3000, 2, 2), (130, 2500, 4, 1)])
def test_groups_of_queries_against_a_long_cache(dev, nq, nk, H, KV):
    """More rows than are shared out over their keys, each list long."""
    _case(1, nq, nk, H, KV, 64, BF16, right=0)
    _case(2, nq, nk, H, KV, 32, F16, F32, lens=[nk, nk // 2 + 7], left=nk - 300, right=0, sinks=5)


def test_output_in_the_place_of_the_queries(dev):
    """Every form: a tile of rows, few rows, keys shared out; rows that are computed again read their query first."""
    import mbrt

    for nq, nk, kw in ((150, 150, dict(left=30, right=0)), (3, 60, dict()), (2, 6000, dict(right=0))):
        say(f"in place nq={nq} nk={nk}")
        q, k, v = _qkv(6, 2, nq, nk, 4, 2, 64, BF16)
        v[0, nk - 2, 0, 5] = float("nan")
        want = mbrt.attention_window(q, k, v, **kw)
        got = mbrt.attention_window(q, k, v, q, **kw)
        assert got is q and torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
