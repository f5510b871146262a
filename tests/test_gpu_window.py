"""flash_attn_window against float64: prompts, single tokens, every mask, with
lengths, sinks, shared heads, strides and rows that see nothing.

Tolerance of o (u = eps / 2 of the type, n keys seen): P is rounded to the type,
each p v off by u p |v|, and l is a sum of unrounded p: at most u sum p |v|
(all roundings in one direction); fp32 scores are off by at most (D + 2) 2^-24
sum |q k| scale, which changes p by that relative amount: a further
2 (D + 2) 2^-24 max_j(sum |q k|) scale sum p |v|; the accumulation n 2^-24; o's
rounding u |o|.  A subnormal P (float16 below 2^-14 of 2^8 times the largest) is
off by 2^-25 instead: n 2^-25 max |v| more.  lse: the scores' error, and
(n + 8) 2^-24 of the sum, plus 2^-22 |lse| + 2^-21 of the logarithm and its scaling.
"""
import math

import pytest
import torch

import prism_amd

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def seen_mask(B, Sq, Sk, window, sinks, causal, q_lens, kv_lens, device="cuda"):
    L = torch.full((B, 1, 1), Sk, device=device) if kv_lens is None else kv_lens.long().clamp(0, Sk)[:, None, None]
    n = torch.full((B, 1, 1), Sq, device=device) if q_lens is None else q_lens.long().clamp(0, Sq)[:, None, None]
    i, j = torch.arange(Sq, device=device)[None, :, None], torch.arange(Sk, device=device)[None, None]
    p = i + L - n
    w = 1 << 40 if window is None else window
    if causal:
        m = (j <= p) & ((j > p - w) | (j < sinks))
    else:
        m = ((p - j).abs() < w) | (j < sinks)
    return m & (j < L) & (i < n)


def reference(q, k, v, mask, scale):
    """(o, lse, tolerance of o, tolerance of lse) in float64."""
    B, Hq, Sq, D = q.shape
    Hk, G = k.shape[1], q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    m = mask[:, None]
    # keys that nobody sees may hold anything
    used = mask.any(1)[:, None, :, None]
    k, v = k.masked_fill(~used, 0), v.masked_fill(~used, 0)
    q = q.masked_fill(~mask.any(2)[:, None, :, None], 0)
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~m, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse.isinf(), torch.zeros_like(lse), lse)[..., None]).masked_fill(~m, 0)
    o = p @ v
    e = (q.abs() @ k.abs().transpose(-1, -2) * scale).masked_fill(~m, 0).amax(-1, keepdim=True) * (D + 2) * 2.0 ** -24
    return o, lse, p @ v.abs(), e, v.abs().amax(2, keepdim=True), m.sum(-1, keepdim=True)


def check(q, k, v, window, *, sinks=0, causal=True, q_lens=None, kv_lens=None, sm_scale=None):
    o, lse = prism_amd.flash_attn_window(q, k, v, window, sinks=sinks, causal=causal, q_lens=q_lens, kv_lens=kv_lens,
                                         sm_scale=sm_scale, return_lse=True)
    assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == q.shape[:3]
    mask = seen_mask(q.shape[0], q.shape[2], k.shape[2], window, sinks, causal, q_lens, kv_lens)
    want, wlse, pv, e, vmax, n = reference(q, k, v, mask, q.shape[-1] ** -0.5 if sm_scale is None else sm_scale)
    u = torch.finfo(q.dtype).eps / 2
    n = n.double()
    tol = pv * (u * 1.001 + 2 * e + n * 2.0 ** -24) + u * want.abs() + n * 2.0 ** -25 * vmax * (q.dtype == torch.float16) \
        + torch.finfo(q.dtype).smallest_normal * u
    bad = (o.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((o.double() - want).abs() / tol).nan_to_num(math.inf).max()))
    empty = ~mask.any(2)[:, None].expand_as(lse)
    assert (lse[empty] == -math.inf).all() and (o[empty] == 0).all()
    ltol = (e[..., 0] + (n[..., 0] + 8) * 2.0 ** -24 + wlse.abs() * 2.0 ** -22 + 2.0 ** -21)
    bad = ((lse.double() - wlse).abs() > ltol) & ~empty
    assert not bad.any(), float(((lse.double() - wlse).abs() / ltol)[~empty].max())
    return o, lse


def make(B, Sq, Sk, Hq, Hk, D, dt, seed=0, projected=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    def one(H, S):
        t = torch.randn((B, S, H, D) if projected else (B, H, S, D), generator=g, device="cuda").to(dt)
        return t.transpose(1, 2) if projected else t
    return one(Hq, Sq), one(Hk, Sk), one(Hk, Sk)


PROMPTS = [  # B, Sq, Sk, Hq, Hk, D, window, sinks, causal
    (1, 65, 65, 1, 1, 64, 1, 0, True), (1, 128, 128, 2, 2, 128, 64, 4, True), (2, 200, 200, 4, 2, 64, 37, 3, True),
    (1, 333, 333, 6, 2, 128, 100, 70, True), (1, 500, 500, 2, 1, 128, None, 0, True), (3, 130, 257, 2, 2, 64, 50, 1, True),
    (1, 300, 40, 2, 2, 64, 16, 2, True), (1, 129, 700, 3, 3, 128, 65, 130, True), (2, 70, 70, 5, 5, 64, 5, 300, True),
    (1, 257, 257, 2, 2, 128, 30, 0, False), (2, 200, 300, 4, 4, 64, 64, 5, False), (1, 100, 600, 2, 2, 64, 3, 129, False),
    (1, 400, 400, 8, 1, 128, 128, 64, False), (1, 333, 100, 1, 1, 64, 9, 1, False), (2, 66, 66, 7, 1, 64, None, 0, False),
    (1, 1100, 1100, 1, 1, 64, 257, 4, True), (1, 1280, 1280, 53, 53, 128, 300, 4, True),
    (1, 1100, 1100, 90, 90, 64, 200, 140, False), (2, 100, 3000, 2, 2, 128, 2500, 9, True),
]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: "-".join(str(x) for x in c))
def test_prompts(case, dt):
    B, Sq, Sk, Hq, Hk, D, window, sinks, causal = case
    q, k, v = make(B, Sq, Sk, Hq, Hk, D, DT[dt], seed=Sq + Sk, projected=Sq % 2 == 0)
    check(q, k, v, window, sinks=sinks, causal=causal)


TOKENS = [  # B, Sq, Sk, Hq, Hk, D, window, sinks, causal
    (1, 1, 1, 1, 1, 64, 1, 0, True), (2, 1, 33, 4, 4, 128, 8, 2, True), (3, 1, 1000, 32, 8, 128, 100, 4, True),
    (1, 1, 5000, 8, 1, 64, None, 0, True), (2, 5, 700, 6, 3, 128, 64, 70, True), (1, 3, 2, 4, 2, 64, 9, 0, True),
    (1, 2, 9001, 64, 2, 64, 4097, 33, True), (8, 1, 300, 5, 5, 128, 31, 32, True), (1, 7, 900, 3, 1, 64, 20, 3, False),
    (2, 1, 20000, 16, 2, 128, 9000, 1, True), (1, 13, 450, 3, 1, 128, 33, 0, True), (5, 4, 64, 8, 2, 128, 64, 64, False),
]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", TOKENS, ids=lambda c: "-".join(str(x) for x in c))
def test_single_tokens(case, dt):
    B, Sq, Sk, Hq, Hk, D, window, sinks, causal = case
    q, k, v = make(B, Sq, Sk, Hq, Hk, D, DT[dt], seed=Sq + Sk, projected=Sk % 2 == 0)
    check(q, k, v, window, sinks=sinks, causal=causal)


@pytest.mark.parametrize("Sq", [1, 3, 140])
def test_lengths(Sq):
    """Lengths of zero, one, less than the queries, the whole, and beyond the
    tensors (cut); unused rows hold NaN and infinities."""
    lens = [0, 1, 2, 64, 65, 139, 200, 999, -3]
    B, Sk = len(lens), 200
    q, k, v = make(B, Sq, Sk, 4, 2, 64, torch.bfloat16, seed=5)
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for ql in (None, kv, torch.tensor([1, 0, 5, 7, 140, 2, 3, 1, 0], dtype=torch.int32, device="cuda")):
        for causal in (True, False):
            for window, sinks in ((17, 3), (1, 0), (None, 0), (70, 130)):
                mask = seen_mask(B, Sq, Sk, window, sinks, causal, ql, kv)
                unused = ~mask.any(1)[:, None, :, None]
                k2, v2 = k.masked_fill(unused, math.nan), v.masked_fill(unused, math.inf)
                q2 = q.masked_fill(~mask.any(2)[:, None, :, None], math.nan)
                check(q2, k2, v2, window, sinks=sinks, causal=causal, q_lens=ql, kv_lens=kv)


@pytest.mark.parametrize("case", [
    (1, 300, 300, 4, 2, 64, 40, 3, True), (1, 333, 400, 2, 2, 128, 65, 0, False), (2, 100, 3000, 2, 2, 128, 2500, 9, True),
    (2, 1, 900, 8, 2, 64, 100, 4, True), (1, 6, 5000, 3, 1, 128, 2000, 0, True), (1, 7, 300, 8, 2, 128, 33, 2, False),
], ids=lambda c: "-".join(str(x) for x in c))
@pytest.mark.parametrize("dt", list(DT))
def test_not_finite_values_stay_with_the_rows_that_see_them(case, dt):
    """NaN and infinities in K, V and Q reach the rows that see them, and no other."""
    B, Sq, Sk, Hq, Hk, D, window, sinks, causal = case
    q, k, v = make(B, Sq, Sk, Hq, Hk, D, DT[dt], seed=Sk)
    seen = seen_mask(B, Sq, Sk, window, sinks, causal, None, None)[0]
    first = int(seen[0].nonzero()[-1])   # the first query's last key, the last query's first past the sinks
    last = int(seen[-1].nonzero()[sinks if causal and Sk > window else 0])
    for at, into, value in ((first, v, math.nan), (last, v, math.inf), (first, k, math.nan), (last, v, -math.inf)):
        x = into.clone()
        x[0, 0, at, 5] = value
        k2, v2 = (x, v) if into is k else (k, x)
        # what the other rows give without that key
        heads = torch.arange(Hq, device="cuda") // (Hq // Hk) == 0
        hit = torch.zeros((B, Hq, Sq), dtype=torch.bool, device="cuda")
        hit[0] = heads[:, None] & seen[:, at][None]
        want = prism_amd.flash_attn_window(q, k, v, window, sinks=sinks, causal=causal).float()
        o, lse = prism_amd.flash_attn_window(q, k2, v2, window, sinks=sinks, causal=causal, return_lse=True)
        assert o[~hit].isfinite().all() and lse[~hit].isfinite().all()
        # both roundings of P and o, each at most a step of the largest |v|
        tol = 4 * torch.finfo(q.dtype).eps * v.abs().max().float()
        assert ((o.float() - want).abs()[~hit] <= tol).all()
        got = o[hit]
        if into is k:
            assert got.isnan().all() and lse[hit].isnan().all()
        else:
            others = [c for c in range(D) if c != 5]
            assert not got[:, 5].isfinite().any()
            assert ((o.float() - want).abs()[hit][:, others] <= tol).all() and lse.isfinite().all()
    x = q.clone()
    x[0, 0, Sq // 2, 7] = math.nan
    o = prism_amd.flash_attn_window(x, k, v, window, sinks=sinks, causal=causal)
    assert o[0, 0, Sq // 2].isnan().all()
    o[0, 0, Sq // 2] = 0
    assert o.isfinite().all()


def test_scale_and_large_scores():
    q, k, v = make(1, 150, 150, 2, 2, 64, torch.bfloat16, seed=1)
    for refused in (0.0, -0.3, math.nan):  # (a masked score times the scale has to stay -inf)
        with pytest.raises(ValueError, match="sm_scale"):
            check(q, k, v, 40, sinks=2, sm_scale=refused)
    check(q, k, v, 40, sinks=2, sm_scale=1e-6)
    check(q * 8, k * 8, v, 40, sinks=2)   # scores of hundreds: one key takes all
    check(q[:, :, :1] * 8, k * 8, v, 40, sinks=2)
    # increasing scores: the running maximum moves all the time
    ramp = torch.arange(150, device="cuda", dtype=torch.float32)[None, None, :, None].expand(1, 2, 150, 64) / 64
    check(torch.ones_like(q), ramp.to(q.dtype), v, None, sm_scale=1.0)


def test_strides():
    """Packed projections, odd offsets, broadcast heads, reversed layouts."""
    dt = torch.bfloat16
    qkv = torch.randn(2, 90, 3, 4, 64, device="cuda").to(dt)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    o = prism_amd.flash_attn_window(q, k, v, 20, sinks=2)
    assert torch.equal(o, prism_amd.flash_attn_window(q.contiguous(), k.contiguous(), v.contiguous(), 20, sinks=2))
    assert o.transpose(1, 2).is_contiguous()  # the layout of the projections
    wide = torch.randn(2, 4, 90, 70, device="cuda").to(dt)
    for t in (wide[..., :64], wide[..., 3:67], torch.randn(90, 64, 4, 2, device="cuda").to(dt).permute(3, 2, 0, 1),
              wide[:1, :1, :, :64].expand(2, 4, 90, 64)):
        check(t, t, k, 33, sinks=1)
        check(t[:, :, :2], t, k, 33, sinks=1)


def test_streams_threads_and_graph():
    q, k, v = make(2, 1, 3000, 8, 2, 128, torch.bfloat16, seed=2)
    kv = torch.tensor([2000, 3000], dtype=torch.int32, device="cuda")
    a = (700,)
    kw = dict(sinks=4, kv_lens=kv)
    want = prism_amd.flash_attn_window(q, k, v, *a, **kw)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(prism_amd.flash_attn_window(q, k, v, *a, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = prism_amd.flash_attn_window(q, k, v, *a, **kw)
        graphs.append((g, got))
    for step in range(3):
        q.normal_()
        kv.sub_(100 * step)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = prism_amd.flash_attn_window(q, k, v, *a, **kw)
        assert all(torch.equal(got, want) for _, got in graphs)


def test_empty():
    for shape_q, shape_k in (((0, 2, 5, 64), (0, 2, 5, 64)), ((1, 2, 0, 64), (1, 2, 5, 64)), ((2, 2, 90, 64), (2, 1, 0, 64)),
                             ((2, 2, 1, 64), (2, 1, 0, 64))):
        q = torch.randn(shape_q, device="cuda").to(torch.bfloat16)
        k = torch.randn(shape_k, device="cuda").to(torch.bfloat16)
        o = prism_amd.flash_attn_window(q, k, k, 3)
        assert o.shape == q.shape and (o == 0).all()
