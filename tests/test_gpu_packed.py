"""flash_attn_packed against float64, forward and backward: packed sequences of many
lengths (none, one, long), keys of their own rows, shared heads, layouts, rows of no
sequence, work lists with and without cuts; values that are not finite; bits that do
not vary.

Tolerances as derived in test_gpu_window.py and test_gpu_window_bwd.py (u = eps / 2 of
the type), but for delta = do . (o + rest): the two hold o's sum to u^2, so what that
leaves off is (u^2 + 2 D 2^-24) sum |do o|; and that sum was made from P rounded to the
type, each P_j off by u P_j at most, which moves do . o by u sum_j P_j |do . v_j|.
"""
import math

import pytest
import torch

import prism_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def cu(lens, first=0):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)


def seen_mask(Tq, Tk, q_bounds, k_bounds, causal):
    m = torch.zeros(Tq, Tk, dtype=torch.bool, device=DEV)
    qb, kb = ([min(max(x, 0), T) for x in b.tolist()] for b, T in ((q_bounds, Tq), (k_bounds, Tk)))
    for a, b, c, d in zip(qb, qb[1:], kb, kb[1:]):
        n, L = b - a, d - c
        i, j = torch.arange(n, device=DEV)[:, None], torch.arange(L, device=DEV)[None]
        m[a:b, c:d] = (j <= i + L - n) if causal else True
    return m


def check(q, k, v, q_bounds, k_bounds=None, *, causal=True, sm_scale=None, do=None):
    Tq, Hq, D = q.shape
    Tk, Hk = k.shape[:2]
    G, scale = Hq // Hk, D ** -0.5 if sm_scale is None else sm_scale
    leaves = [t.detach().requires_grad_(do is not None) for t in (q, k, v)]
    o, lse = prism_amd.flash_attn_packed(*leaves, q_bounds, cu_seqlens_k=k_bounds, causal=causal, sm_scale=sm_scale,
                                         return_lse=True)
    assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (Hq, Tq)
    if Tk == 0:  # (nothing for the products below)
        assert not o.any() and (lse == -math.inf).all()
        assert do is None or not any(g.any() for g in torch.autograd.grad(o, leaves, do))
        return o, lse
    mask = seen_mask(Tq, Tk, q_bounds, q_bounds if k_bounds is None else k_bounds, causal)
    rows, keys = mask.any(1)[:, None], mask.any(0)[:, None]
    heads = lambda t, live: t.double().transpose(0, 1).masked_fill(~live, 0)  # noqa: E731
    q64, k64, v64 = heads(q, rows), *(heads(t, keys).repeat_interleave(G, 0) for t in (k, v))
    x = (q64 @ k64.transpose(1, 2).contiguous() * scale).masked_fill(~mask, -math.inf)
    want_lse = torch.logsumexp(x, -1)
    P = torch.exp(x - want_lse.nan_to_num(neginf=0.0)[..., None])
    o64 = P @ v64
    u, n = torch.finfo(q.dtype).eps / 2, mask.sum(1).double()[None, :, None]
    half, small = q.dtype == torch.float16, torch.finfo(q.dtype).smallest_normal
    sizes = (q64.abs() @ k64.abs().transpose(1, 2).contiguous() * scale).masked_fill(~mask, 0).amax(-1, keepdim=True)
    e = sizes * (D + 2) * 2.0 ** -24
    tol = (P @ v64.abs()) * (u * 1.001 + 2 * e + n * 2.0 ** -24) + u * o64.abs() + small * u \
        + n * 2.0 ** -25 * v64.abs().amax(1, keepdim=True) * half
    worst = ((o.detach().double().transpose(0, 1) - o64).abs() / tol).nan_to_num(math.inf).max().item() if o.numel() else 0
    assert worst <= 1, f"o: {worst:.3f} of the bound"
    none = ~mask.any(1)
    assert (o[none] == 0).all() and (lse[:, none] == -math.inf).all()
    ltol = e[..., 0] + (n[..., 0] + 8) * 2.0 ** -24 + want_lse.abs() * 2.0 ** -22 + 2.0 ** -21
    assert ((lse.double() - want_lse).abs() <= ltol)[:, ~none].all()
    if do is None:
        return o, lse
    got = torch.autograd.grad(o, leaves, do)
    do64 = heads(do, rows)
    dP = do64 @ v64.transpose(1, 2).contiguous()
    dS = P * (dP - (do64 * o64).sum(-1, keepdim=True))
    tr = lambda a, b: (a.transpose(1, 2).contiguous() @ b).view(Hk, G, Tk, D).sum(1)  # noqa: E731
    want = [scale * (dS @ k64), scale * tr(dS, q64), tr(P, do64)]
    N = float(max(Tk, Tq * G)) * 2.0 ** -24
    r = 4 * e
    d2 = (do64.abs() @ v64.abs().transpose(1, 2).contiguous()).masked_fill(~mask, 0).amax(-1, keepdim=True)
    sub = 2.0 ** -25 * mask * half
    d0 = (u * u + 2 * D * 2.0 ** -24) * (do64 * o64).abs().sum(-1, keepdim=True) \
        + u * (P * dP.abs()).sum(-1, keepdim=True)
    ds = P * (d0 + (r + 1.01 * u) * (dP - (do64 * o64).sum(-1, keepdim=True)).abs() + 2.0 ** -24 * (D + n) * d2) + sub
    dp = P * (u * 1.01 + r) + sub
    tols = [scale * (ds @ k64.abs() + N * (dS.abs() @ k64.abs())), scale * (tr(ds, q64.abs()) + N * tr(dS.abs(), q64.abs())),
            tr(dp, do64.abs()) + N * tr(P, do64.abs())]
    for name, a, b, t in zip(("dq", "dk", "dv"), got, want, tols):
        assert a.dtype == q.dtype
        t = t + u * b.abs() + small * u
        worst = ((a.double().transpose(0, 1) - b).abs() / t).nan_to_num(math.inf).max().item() if a.numel() else 0
        assert worst <= 1, f"{name}: {worst:.3f} of the bound"
    assert (got[0][none] == 0).all() and (got[1][~keys[:, 0]] == 0).all() and (got[2][~keys[:, 0]] == 0).all()
    return (o.detach(), lse, *got)


def make(T, H, D, dt, seed, layout="dense"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if layout == "heads":  # [H, T, D] in memory
        return torch.randn(H, T, D, generator=g, device=DEV).to(dt).transpose(0, 1)
    if layout == "wide":   # part of a projection's output
        return torch.randn(T, 3 * H, D, generator=g, device=DEV).to(dt)[:, H:2 * H]
    if layout == "odd":    # rows that are not 16-byte aligned
        return torch.randn(T, H, D + 1, generator=g, device=DEV).to(dt)[..., 1:]
    return torch.randn(T, H, D, generator=g, device=DEV).to(dt)


CASES = [  # lengths, Hq, Hk, D, causal, layout
    ([1], 1, 1, 64, True, "dense"), ([0, 1, 0, 2, 0], 4, 2, 128, True, "dense"), ([63, 64, 65], 2, 2, 64, True, "heads"),
    ([5, 300, 1, 129, 40], 6, 2, 128, True, "wide"), ([200, 31], 8, 1, 64, True, "odd"), ([17, 90, 33], 5, 5, 128, False, "dense"),
    ([400, 3, 150], 4, 1, 64, False, "heads"), ([700], 2, 1, 128, True, "dense"), ([1100, 0, 700, 64], 2, 2, 64, True, "wide"),
    ([1500, 200], 4, 2, 128, True, "dense"), ([128, 1000, 900], 3, 1, 128, False, "dense"),
    ([3, 9, 0, 1, 14, 2] * 30, 4, 2, 64, True, "dense"), ([2, 0, 25, 1] * 40 + [600], 2, 1, 128, True, "heads"),
    ([2500], 1, 1, 64, True, "dense"), ([40] * 60, 7, 1, 64, True, "dense"),
]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-" + "-".join(str(x) for x in c[1:]))
def test_sequences(case, dt):
    lens, Hq, Hk, D, causal, layout = case
    T = sum(lens)
    q, k, v, do = (make(T, H, D, DT[dt], s, layout) for s, H in enumerate((Hq, Hk, Hk, Hq)))
    a = check(q, k, v, cu(lens), causal=causal, do=do)
    if layout != "odd":
        if layout == "heads":
            assert a[0].stride() == q.stride() and a[2].stride() == q.stride()
    b = check(q, k, v, cu(lens), causal=causal, do=do)
    assert all(torch.equal(x, y) for x, y in zip(a, b))  # the same bits every time
    with torch.no_grad():
        assert torch.equal(prism_amd.flash_attn_packed(q, k, v, cu(lens), causal=causal), a[0])


KEYS = [  # queries, keys of the sequences
    ([1, 1, 1], [40, 1, 700]), ([5, 0, 64, 3], [5, 30, 200, 1]), ([100, 33], [600, 33]), ([70], [0]), ([0, 40], [90, 41]),
    ([130, 2], [64, 900]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", KEYS, ids=lambda c: f"{c[0]}-{c[1]}".replace(" ", ""))
def test_keys_of_their_own(case, causal):
    for D, dt in ((64, torch.bfloat16), (128, torch.float16)):
        q, do = (make(sum(case[0]), 4, D, dt, s) for s in (1, 2))
        k, v = (make(sum(case[1]), 2, D, dt, s) for s in (3, 4))
        check(q, k, v, cu(case[0]), cu(case[1]), causal=causal, do=do, sm_scale=0.2)


@pytest.mark.parametrize("many", [False, True])
def test_rows_of_no_sequence(many):
    """Rows before the first sequence and behind the last, which hold NaN: 0, no
    gradients, and not read; bounds outside the tensors are cut to them."""
    lens = [40, 0, 130, 7] + ([3] * 70 if many else [])
    T = sum(lens) + 45 + 300
    q, k, v, do = (make(T, H, 64, torch.bfloat16, s) for s, H in enumerate((4, 2, 2, 4)))
    for t in (q, k, v, do):
        t[:45] = float("nan")
        t[45 + sum(lens):] = float("inf")
    check(q, k, v, cu(lens, 45), do=do)
    check(q, k, v, cu(lens, 45), causal=False, do=do)
    for t in (q, k, v, do):
        t[:45] = 0.5
        t[45 + sum(lens):] = 0.25
    b = cu(lens, 45)
    b[0], b[-1] = -7, T + 99
    check(q, k, v, b, do=do)


def test_more_list_tiles_times_parts_than_32_bits():
    """2^28 keys (one row, at stride 0) cut into a thousand parts, all seen by a few rows: with
    k = 0 and small integers in v every sum of a part is exact, so o is v itself."""
    n, D = 1 << 28, 64
    q = make(3, 1, D, torch.bfloat16, 1)
    k = torch.zeros(1, 1, D, dtype=torch.bfloat16, device=DEV)
    v = torch.randint(-4, 5, (1, 1, D), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).bfloat16()
    o, lse = prism_amd.flash_attn_packed(q, k.expand(n, 1, D), v.expand(n, 1, D), cu([3]), cu_seqlens_k=cu([n]), causal=False,
                                         return_lse=True)
    assert torch.equal(o, v.expand(3, 1, D)) and ((lse - 28 * math.log(2)).abs() <= 28 * 2.0 ** -22).all()


@pytest.mark.parametrize("B", [5, 61, 700])
def test_bounds_that_decrease_stay_inside(B):
    """Bounds in any order: what comes of them is not defined, but the calls before and
    after, and tensors beside theirs, are as they were."""
    T, H, D = 1500, 2, 64
    pool = torch.full((4, T, H, D), 3.0, dtype=torch.bfloat16, device=DEV)
    pool[1:3] = make(2 * T, H, D, torch.bfloat16, 3).view(2, T, H, D)
    q, k = (x.detach().requires_grad_(True) for x in pool[1:3])
    good = cu([700, 300, 500])
    want, _ = prism_amd.flash_attn_packed(q, k, k, good, return_lse=True)
    for seed in range(3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        any_, other = (torch.randint(-99, T + 99, (B + 1,), generator=g, device=DEV, dtype=torch.int32) for _ in "qk")
        for causal in (True, False):
            o = prism_amd.flash_attn_packed(q, k, k, any_, cu_seqlens_k=other, causal=causal)
            torch.autograd.grad(o, (q, k), torch.ones_like(o))
    assert torch.equal(want, prism_amd.flash_attn_packed(q, k, k, good))
    assert (pool[0] == 3).all() and (pool[3] == 3).all()


def test_no_tokens_and_no_sequences():
    z = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.randn(9, 4, 64, device=DEV).bfloat16().requires_grad_(True)
    k = torch.randn(9, 2, 64, device=DEV).bfloat16().requires_grad_(True)
    o, lse = prism_amd.flash_attn_packed(q, k, k, z, return_lse=True)
    dq, dk = torch.autograd.grad(o, (q, k), torch.ones_like(o))
    assert not o.any() and (lse == -math.inf).all() and not dq.any() and not dk.any()
    for Tq, Tk in ((0, 9), (9, 0), (0, 0)):
        qs, ks = q.detach()[:Tq].requires_grad_(True), k.detach()[:Tk].requires_grad_(True)
        o = prism_amd.flash_attn_packed(qs, ks, ks, torch.tensor([0, Tq], dtype=torch.int32, device=DEV),
                                        cu_seqlens_k=torch.tensor([0, Tk], dtype=torch.int32, device=DEV))
        dq, dk = torch.autograd.grad(o, (qs, ks), torch.ones_like(o))
        assert o.shape == (Tq, 4, 64) and not o.any() and not dq.any() and not dk.any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[100, 40], [900, 300]])
def test_not_finite_reaches_who_sees_it(lens, D):
    T = sum(lens)
    for dt in (torch.bfloat16, torch.float16):
        q, k, v = (make(T, H, D, dt, s) for s, H in enumerate((4, 2, 2)))
        want, _ = check(q, k, v, cu(lens))
        place = lens[0] - 23
        for t, bad in ((v, float("nan")), (v, float("inf")), (k, float("nan"))):
            x = t.clone()
            x[place, 1, 5] = bad
            o = prism_amd.flash_attn_packed(q, x if t is k else k, x if t is v else v, cu(lens))
            hit = torch.zeros(T, 4, dtype=torch.bool, device=DEV)
            hit[place:lens[0], 2:] = True
            # (rows of a wave that holds such a value are added up key by key: as near to
            # float64 as the others, not the same bits)
            assert torch.isfinite(o[~hit]).all() and not torch.isfinite(o[..., 5][hit]).any()
            assert torch.allclose(o[~hit].float(), want[~hit].float(), rtol=2 ** -6, atol=2 ** -7)


def test_gradients_against_differences():
    lens = [5, 11]
    q, k, v = (make(16, H, 64, torch.float16, s) for s, H in enumerate((2, 1, 1)))
    c = torch.randn(16, 2, 64, device=DEV, dtype=torch.float64)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(prism_amd.flash_attn_packed(*leaves, cu(lens)), leaves, c.half())
    f = lambda *t: (prism_amd.flash_attn_packed(*t, cu(lens)).double() * c.half().double()).sum().item()  # noqa: E731
    for x, g in enumerate(grads):
        for seed in range(4):
            e = make(16, leaves[x].shape[1], 64, torch.float16, 50 + seed).double()
            h = 2.0 ** -5
            a, b = ([t if y != x else (t.double() + s * h * e).half() for y, t in enumerate((q, k, v))] for s in (1, -1))
            step = (a[x].double() - b[x].double())  # (what float16 makes of it)
            want = (g.double() * step).sum().item()
            # o's rounding: 2,048 values of size 1, 2^-11 each, random; P's likewise; h^3 of the third derivative
            assert abs(f(*a) - f(*b) - want) <= 2 * 2048 ** 0.5 * 2.0 ** -11 * 4 + 100 * h ** 3 + 0.02 * abs(want)


def test_is_what_padding_gives():
    """The same sequences through flash_attn_window, padded."""
    lens = [37, 500, 128]
    T, N = sum(lens), max(lens)
    q, k, v = (make(T, H, 128, torch.bfloat16, s) for s, H in enumerate((8, 2, 2)))
    o = prism_amd.flash_attn_packed(q, k, v, cu(lens))
    pad = lambda t: torch.nn.utils.rnn.pad_sequence(t.split(lens), batch_first=True).transpose(1, 2).contiguous()  # noqa: E731
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    w = prism_amd.flash_attn_window(pad(q), pad(k), pad(v), None, q_lens=n, kv_lens=n).transpose(1, 2)
    w = torch.cat([w[b, :m] for b, m in enumerate(lens)])
    assert N == 500 and torch.allclose(o.float(), w.float(), rtol=2 ** -7, atol=2 ** -8)
