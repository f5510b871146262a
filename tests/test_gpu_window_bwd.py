"""Gradients of flash_attn_window against float64 and against differences.

Tolerance (u = eps / 2 of the type): with exact P, dP, delta,
  o is stored rounded, so delta is off by u sum |do o|, dS = P (dP - delta) by P
  times that; P itself by a relative r = 4 e, e = (D + 2) 2^-24 max (sum |q k|)
  scale (scores, lse); dP by D 2^-24 sum |do v|; dS and P are rounded to the
  type (u).  So |ddS| <= P (u D1 + (r + u) |dP - delta| + 2^-24 (D + n) D2), D1 = sum
  |do o|, D2 = max sum |do v|; dq and dk are off by scale times the products
  of that bound with |k| and |q|, dv by (u + r) P^T |do|, each by its own
  rounding u |.| and fp32 sums of N terms (N 2^-24 of the terms).  float16
  adds its subnormal steps: 2^-25 for each P and dS, times |do|, |k|, |q|.
Where rows see 64 keys at most (few), delta is the sum of P dP: r sum P |dP| in
the place of u D1.
"""
import math

import pytest
import torch

import prism_amd
from tests.test_gpu_window import DT, make, seen_mask
from tests.test_gpu_window import check as check_forward

pytestmark = pytest.mark.gpu


def check(q, k, v, do, window, *, sinks=0, causal=True, q_lens=None, kv_lens=None, sm_scale=None, few=False):
    B, Hq, Sq, D = q.shape
    Hk, Sk, G = k.shape[1], k.shape[2], Hq // k.shape[1]
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = prism_amd.flash_attn_window(*leaves, window, sinks=sinks, causal=causal, q_lens=q_lens, kv_lens=kv_lens,
                                    sm_scale=sm_scale)
    got = torch.autograd.grad(o, leaves, do)
    scale = D ** -0.5 if sm_scale is None else sm_scale
    mask = seen_mask(B, Sq, Sk, window, sinks, causal, q_lens, kv_lens)
    rows, keys = mask.any(2)[:, None, :, None], mask.any(1)[:, None, :, None]
    q64, do64 = q.double().masked_fill(~rows, 0), do.double().masked_fill(~rows, 0)
    k64, v64 = (t.double().masked_fill(~keys, 0).repeat_interleave(G, 1) for t in (k, v))
    m = mask[:, None]
    x = (q64 @ k64.transpose(-1, -2) * scale).masked_fill(~m, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top.isinf(), torch.zeros_like(top), top))
    P = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    o64 = P @ v64
    dP = do64 @ v64.transpose(-1, -2)
    delta = (do64 * o64).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    share = lambda t: t.view(B, Hk, G, Sk, D).sum(2)  # noqa: E731
    tr = lambda a, b: share(a.transpose(-1, -2).contiguous() @ b)  # noqa: E731
    want = [scale * (dS @ k64), scale * tr(dS, q64), tr(P, do64)]
    # the bound above
    u, n = torch.finfo(q.dtype).eps / 2, float(max(Sk, Sq * G))
    r = 4 * (D + 2) * 2.0 ** -24 * (q64.abs() @ k64.abs().transpose(-1, -2) * scale).masked_fill(~m, 0).amax(-1, keepdim=True)
    d1 = (do64 * o64).abs().sum(-1, keepdim=True)
    d2 = (do64.abs() @ v64.abs().transpose(-1, -2)).masked_fill(~m, 0).amax(-1, keepdim=True)
    sub = 2.0 ** -25 * m * (q.dtype == torch.float16)
    d0 = r * (P * dP.abs()).sum(-1, keepdim=True) if few else u * d1
    ds = P * (d0 + (r + 1.01 * u) * (dP - delta).abs() + 2.0 ** -24 * (D + n) * d2) + sub
    dp = P * (u * 1.01 + r) + sub
    N = n * 2.0 ** -24
    tols = [scale * (ds @ k64.abs() + N * (dS.abs() @ k64.abs())), scale * (tr(ds, q64.abs()) + N * tr(dS.abs(), q64.abs())),
            tr(dp, do64.abs()) + N * tr(P, do64.abs())]
    for name, a, b, t in zip(("dq", "dk", "dv"), got, want, tols):
        assert a.shape == b.shape and a.dtype == q.dtype
        t = t + u * b.abs() + torch.finfo(q.dtype).smallest_normal * u
        bad = ~((a.double() - b).abs() <= t)
        assert not bad.any(), (name, int(bad.sum()), float(((a.double() - b).abs() / t).nan_to_num(math.inf).max()))
    assert (got[0][~rows.expand_as(got[0])] == 0).all()
    assert (got[1][~keys.expand_as(got[1])] == 0).all() and (got[2][~keys.expand_as(got[2])] == 0).all()
    return got


CASES = [  # B, Sq, Sk, Hq, Hk, D, window, sinks, causal
    (1, 1, 1, 1, 1, 64, 1, 0, True), (2, 1, 40, 4, 2, 128, 8, 2, True), (1, 65, 65, 1, 1, 64, 1, 0, True),
    (1, 128, 128, 2, 2, 128, 64, 4, True), (2, 200, 200, 4, 2, 64, 37, 3, True), (1, 333, 333, 6, 2, 128, 100, 70, True),
    (1, 500, 500, 2, 1, 128, None, 0, True), (3, 130, 257, 2, 2, 64, 50, 1, True), (1, 300, 40, 2, 2, 64, 16, 2, True),
    (1, 129, 700, 3, 3, 128, 65, 130, True), (2, 70, 70, 5, 5, 64, 5, 300, True), (1, 257, 257, 2, 2, 128, 30, 0, False),
    (2, 200, 300, 4, 4, 64, 64, 5, False), (1, 100, 600, 2, 2, 64, 3, 129, False), (1, 400, 400, 8, 1, 128, 128, 64, False),
    (1, 333, 100, 1, 1, 64, 9, 1, False), (2, 66, 66, 7, 1, 64, None, 0, False), (1, 1500, 1500, 8, 1, 64, 40, 4, True),
    (1, 1300, 1300, 2, 1, 128, 700, 150, False), (1, 2000, 2000, 4, 2, 128, None, 0, True),
    # more tiles than the chip holds at once, and a few over: the last round is cut
    (1, 1280, 1280, 53, 53, 128, 300, 4, True), (1, 1100, 1100, 90, 90, 64, 200, 140, False),
]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_against_float64(case, dt):
    B, Sq, Sk, Hq, Hk, D, window, sinks, causal = case
    q, k, v = make(B, Sq, Sk, Hq, Hk, D, DT[dt], seed=Sq + Sk, projected=Sq % 2 == 0)
    do = torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(q.dtype)
    a = check(q, k, v, do, window, sinks=sinks, causal=causal)
    b = check(q, k, v, do, window, sinks=sinks, causal=causal)
    assert all(torch.equal(x, y) for x, y in zip(a, b))  # the same bits every time


@pytest.mark.parametrize("Sq", [1, 140])
def test_lengths(Sq):
    """Lengths of zero, one, less than the queries, beyond the tensors; unused
    rows of q, k, v and do hold NaN and infinities."""
    lens = [0, 1, 2, 64, 65, 139, 200, 999, -3]
    B, Sk = len(lens), 200
    q, k, v = make(B, Sq, Sk, 4, 2, 64, torch.bfloat16, seed=5)
    do = make(B, Sq, Sk, 4, 2, 64, torch.bfloat16, seed=6)[0]
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for ql in (None, kv, torch.tensor([1, 0, 5, 7, 140, 2, 3, 1, 0], dtype=torch.int32, device="cuda")):
        for causal in (True, False):
            for window, sinks in ((17, 3), (1, 0), (None, 0), (70, 130)):
                mask = seen_mask(B, Sq, Sk, window, sinks, causal, ql, kv)
                keys, rows = ~mask.any(1)[:, None, :, None], ~mask.any(2)[:, None, :, None]
                check(q.masked_fill(rows, math.nan), k.masked_fill(keys, math.nan), v.masked_fill(keys, math.inf),
                      do.masked_fill(rows, math.nan), window, sinks=sinks, causal=causal, q_lens=ql, kv_lens=kv)


def test_by_differences():
    """Directional derivative of a weighted sum of o, averaged over a step large
    against bfloat16's rounding of o."""
    q, k, v = make(1, 96, 96, 4, 2, 64, torch.float16, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randn(q.shape, generator=g, device="cuda").half()
    dirs = [torch.randn(t.shape, generator=g, device="cuda") for t in (q, k, v)]
    f = lambda s: float((prism_amd.flash_attn_window(  # noqa: E731
        *[(t.float() + s * d).half() for t, d in zip((q, k, v), dirs)], 40, sinks=3).double() * w.double()).sum())
    e = 2.0 ** -5
    diff = (f(e) - f(-e)) / (2 * e)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(prism_amd.flash_attn_window(*leaves, 40, sinks=3), leaves, w)
    want = sum(float((a.double() * d.double()).sum()) for a, d in zip(grads, dirs))
    # 24,576 outputs of size ~0.3, each off by 2^-11 relative at either end, weights ~1, random signs:
    # sqrt(2 * 24576) 0.3 2^-11 / (2 e) ~ 0.5; inputs rounded after the step: as much again three times;
    # third derivatives e^2 / 6 of terms ~ 1 each: sqrt(24576) e^2 ~ 0.15.  Twice their sum.
    assert abs(diff - want) <= 2 * (4 * 0.5 + 0.15), (diff, want)


def test_layouts_broadcasts_and_partial_leaves():
    dt = torch.bfloat16
    qkv = torch.randn(2, 90, 3, 4, 64, device="cuda").to(dt).requires_grad_(True)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    do = torch.randn(2, 4, 90, 64, device="cuda").to(dt)
    (packed,) = torch.autograd.grad(prism_amd.flash_attn_window(q, k, v, 20, sinks=2), qkv, do)
    parts = check(q.detach().contiguous(), k.detach().contiguous(), v.detach().contiguous(), do, 20, sinks=2)
    for i, t in enumerate(parts):
        assert torch.equal(packed[:, :, i].transpose(1, 2), t)
    # one key head expanded over four: its gradient is their sum
    one = torch.randn(2, 1, 90, 64, device="cuda").to(dt).requires_grad_(True)
    o = prism_amd.flash_attn_window(q.detach(), one.expand(2, 4, 90, 64), v.detach(), 20, sinks=2)
    (wide,) = torch.autograd.grad(o, one, do)
    full = check(q.detach(), one.detach().expand(2, 4, 90, 64), v.detach(), do, 20, sinks=2)[1]
    assert torch.equal(wide, full.sum(1, keepdim=True))
    # gradient that arrives broadcast, and leaves that need none
    x = k.detach().requires_grad_(True)
    o = prism_amd.flash_attn_window(q.detach(), x, v.detach(), 20)
    (g1,) = torch.autograd.grad(o.sum(), x)
    assert torch.equal(g1, check(q.detach(), k.detach(), v.detach(), torch.ones_like(o), 20)[1])


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", [(3, 5, 5, 8, 2, 64, None, 0, True), (2, 64, 64, 4, 2, 128, None, 0, False),
                                  (2, 300, 300, 4, 2, 64, 3, 0, True), (1, 200, 333, 6, 2, 128, 40, 24, True),
                                  (2, 150, 150, 5, 5, 64, 30, 5, False), (1, 300, 300, 40, 1, 128, 60, 4, True),
                                  (2, 700, 40, 7, 1, 64, 9, 0, True), (1, 2000, 2000, 33, 33, 64, 12, 2, True)],
                         ids=lambda c: "-".join(str(x) for x in c))
def test_few_keys_with_a_common_part(case, dt):
    """Values that share a large part (64, times do of one sign): the rounding of o
    in delta would be far larger than dS, which does not depend on that part."""
    B, Sq, Sk, Hq, Hk, D, window, sinks, causal = case
    q, k, v = make(B, Sq, Sk, Hq, Hk, D, DT[dt], seed=Sq + Sk)
    do = torch.randn_like(q).abs()
    lens = torch.tensor([Sk, Sk // 2, 1], dtype=torch.int32, device="cuda")[:B]
    for n in (None, lens):
        check(q, k, v + 64, do, window, sinks=sinks, causal=causal, kv_lens=n, q_lens=n if Sq == Sk else None, few=True)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", [(2, 300, 300, 4, 2, 64, 100, 0, True), (1, 130, 900, 2, 2, 128, None, 0, True),
                                  (1, 3, 2000, 8, 2, 64, 500, 9, True), (2, 1, 70, 4, 1, 128, None, 0, True),
                                  (1, 300, 300, 40, 1, 128, 66, 4, False), (1, 1300, 1300, 2, 1, 128, 700, 150, False)],
                         ids=lambda c: "-".join(str(x) for x in c))
def test_rest_of_the_rounding(case, dt):
    """o + rest is o unrounded: off by the products' roundings only where P is exact
    (equal scores of a power of two of keys), and what o stands for elsewhere."""
    B, Sq, Sk, Hq, Hk, D, window, sinks, causal = case
    q, k, v = make(B, Sq, Sk, Hq, Hk, D, DT[dt], seed=Sq + Sk)
    w = 1 << 29 if window is None else window
    o, lse, rest = prism_amd.ops.window_fwd(q, k, v, w, sinks, causal, None, None, D ** -0.5, True, True)
    o2, lse2 = prism_amd.ops.window_fwd(q, k, v, w, sinks, causal, None, None, D ** -0.5, True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2) and rest.stride() == o.stride() and rest.dtype == o.dtype
    u = torch.finfo(o.dtype).eps / 2
    assert (rest.float().abs() <= u * o.float().abs() * (1 + u) + 2.0 ** -25).all()
    # equal scores: o is the mean of the seen values, P = 1 exactly
    flat = torch.zeros_like(q)
    o, _, rest = prism_amd.ops.window_fwd(flat, k, v, w, sinks, causal, None, None, D ** -0.5, False, True)
    m = seen_mask(B, Sq, Sk, window, sinks, causal, None, None)[:, None].double()
    n = m.sum(-1, keepdim=True)
    mean = (m @ v.double().repeat_interleave(Hq // Hk, 1)) / n.clamp(min=1)
    size = (m @ v.double().abs().repeat_interleave(Hq // Hk, 1)) / n.clamp(min=1)
    # fp32 sums of n terms, the division, rest's own rounding (fp16: its subnormal step)
    tol = (n + 4) * 2.0 ** -24 * size + u * u * mean.abs() * 1.01 + 2.0 ** -25 * (dt == "fp16")
    assert ((o.double() + rest.double() - mean).abs() <= tol).all()


RAGGED = [  # B, S, Hq, Hk, D, window, sinks, causal: a round or two of tiles, sequences of their own lengths
    (5, 1000, 8, 4, 64, 200, 70, True), (5, 1000, 7, 7, 128, 300, 4, False), (3, 1000, 16, 2, 128, 300, 0, True),
    (64, 100, 8, 8, 64, 30, 4, True), (65, 100, 8, 8, 64, 30, 4, True), (33, 130, 9, 9, 128, None, 0, True),
    (2, 2500, 8, 8, 64, 400, 140, False),
]


@pytest.mark.parametrize("case", RAGGED, ids=lambda c: "-".join(str(x) for x in c))
def test_ragged_batches(case):
    """Tiles taken by rank over sequences of different lengths (zero, one, all)."""
    B, S, Hq, Hk, D, window, sinks, causal = case
    q, k, v = make(B, S, S, Hq, Hk, D, torch.bfloat16, seed=S + B, projected=True)
    do = torch.randn_like(q)
    lens = torch.tensor([S, 0, S // 2 + 37, 64, S - 1, 1] * (B // 6 + 1), dtype=torch.int32, device="cuda")[:B]
    other = lens.flip(0).contiguous()
    for ql, kv in ((lens, lens), (other, lens), (lens, None), (None, lens)):
        mask = seen_mask(B, S, S, window, sinks, causal, ql, kv)
        rows, keys = ~mask.any(2)[:, None, :, None], ~mask.any(1)[:, None, :, None]
        kw = dict(sinks=sinks, causal=causal, q_lens=ql, kv_lens=kv)
        args = (q.masked_fill(rows, math.nan), k.masked_fill(keys, math.nan), v.masked_fill(keys, math.inf))
        check_forward(*args, window, **kw)
        check(*args, do.masked_fill(rows, math.nan), window, **kw)


def test_captured():
    q, k, v = make(2, 300, 300, 4, 2, 64, torch.bfloat16, seed=2)
    do = torch.randn_like(q)
    n = torch.tensor([300, 200], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        return torch.autograd.grad(prism_amd.flash_attn_window(*leaves, 50, sinks=70, q_lens=n, kv_lens=n), leaves, do)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            for t in leaves:
                t.normal_()
            n.sub_(30)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_empty():
    for sq, sk in ((0, 5), (5, 0), (0, 0)):
        q = torch.randn(2, 2, sq, 64, device="cuda").half().requires_grad_(True)
        k = torch.randn(2, 1, sk, 64, device="cuda").half().requires_grad_(True)
        v = k.detach().clone().requires_grad_(True)
        grads = torch.autograd.grad(prism_amd.flash_attn_window(q, k, v, 3).sum(), (q, k, v))
        assert all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, (q, k, v)))


def test_opcheck():
    q, k, v = make(1, 70, 70, 2, 1, 64, torch.bfloat16)
    n = torch.tensor([50], dtype=torch.int32, device="cuda")
    torch.library.opcheck(torch.ops.prism.window_fwd.default, (q, k, v, 9, 2, True, n, n, 0.1, True, True),
                          test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.prism.window_fwd.default, (q, k, v, 9, 2, True, n, n, 0.1, False, False),
                          test_utils=("test_schema", "test_faketensor"))
    o, lse, rest = torch.ops.prism.window_fwd(q, k, v, 9, 2, True, n, n, 0.1, True, True)
    torch.library.opcheck(torch.ops.prism.window_bwd.default, (q, q, k, v, o, rest, lse, 9, 2, True, n, None, 0.1),
                          test_utils=("test_schema", "test_faketensor"))
