"""append_paged, gather_paged and flash_attn_paged: the cache's contents bit for bit
against their definition in float64, attention against float64 over the values that the
cache holds; page sizes, lengths, tables with pages that are none, layouts, both widths.

Tolerance of o: as derived in test_gpu_window.py (u = eps / 2 of the type).  Over 4 bits K
and V are exact in the products and P times V's scale is rounded to bfloat16, so P's part
takes bfloat16's u; float16 queries meet K as float16 (values below 2^-14 of K lose up to
2^-25: D 2^-25 max |q| scale in a score).
"""
import math
import random

import pytest
import torch

import prism_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ------------------------------------------------------------------ the definition
def levels_of(x):
    """float64 values that 4 bits hold of x [.., D] (of a 16-bit type), blocks of 32
    channels that are not finite as NaN: the nearest level by comparing all of them."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** -126)
    for e in range(-126, 127):
        scale = torch.where(top > 6 * scale, torch.full_like(scale, 2.0 ** (e + 1)), scale)
    grid = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    far = (b.abs()[..., None] / scale[..., None] - grid).abs()
    near = far.amin(-1, keepdim=True)
    even = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)  # (even codes first: halves go to them)
    code = even[(far[..., even] == near).int().argmax(-1)]
    y = grid[code] * scale * torch.where(torch.signbit(b), -1.0, 1.0)
    return torch.where(torch.isfinite(b).all(-1, keepdim=True), y, torch.full_like(y, math.nan)).flatten(-2)


def of_cache(cache, D):
    """float64 [pages, heads, page size, D] of what a cache holds."""
    if cache.dtype is not torch.uint8:
        return cache.double()
    P, H, n = cache.shape
    page = n // (D // 2 + D // 32)
    code, byte = cache[..., :page * D // 2].reshape(P, H, page, D // 2), cache[..., page * D // 2:].reshape(P, H, page, D // 32)
    pair = torch.stack([code & 15, code >> 4], -1).flatten(-2).long()
    v = torch.tensor(LEVELS + [-x for x in LEVELS], dtype=torch.float64, device=cache.device)[pair]
    s = torch.exp2(byte.double() - 127)
    s[byte == 255] = math.nan
    return v * s.repeat_interleave(32, -1)


def turned(k, at, freqs, interleaved, amplitude, dtype, axis_pairs=None):
    """k [T, H, D] turned at positions [T] (or [T, A]) in float64, rounded to dtype."""
    at = at.double()
    if axis_pairs:
        at = at.repeat_interleave(torch.tensor(axis_pairs, device=k.device), -1)
    else:
        at = at[:, None]
    unit = torch.polar(torch.full((), amplitude, dtype=torch.float64, device=k.device), at * freqs)[:, None]
    R = 2 * freqs.numel()
    x = k.double()
    rot = x[..., :R]
    pair = rot.unflatten(-1, (R // 2, 2)) if interleaved else rot.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit)
    return torch.cat([z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2), x[..., R:]], -1).to(dtype)


def places_of(lens, new):
    """(sequence, place) of every new token."""
    who = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], dtype=torch.long, device=DEV)
    at = torch.tensor([L - n + i for L, n in zip(lens, new) for i in range(n)], dtype=torch.long, device=DEV)
    return who, at


def table_for(lens, page, seed=0, spare=3, wide=None):
    need = [max(0, -(-n // page)) for n in lens]
    pages = sum(need) + spare
    ids = list(range(pages))
    random.Random(seed).shuffle(ids)
    width, rows = max(max(need, default=0), 1) if wide is None else wide, []
    for n in need:
        rows.append(ids[:n] + [-1] * (width - n))
        ids = ids[n:]
    return torch.tensor(rows, dtype=torch.int32, device=DEV).view(len(lens), width), pages


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cu(lens):
    return ints([sum(lens[:i]) for i in range(len(lens) + 1)])


def filled(pages, page, H, D, dtype, bits, seed=0):
    """A cache that holds something everywhere."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    kc, vc = prism_amd.paged_cache(pages, page, H, D, dtype=dtype, bits=bits)
    for c in (kc, vc):
        if bits == 16:
            c.copy_(torch.randn(c.shape, generator=g, device=DEV))
        else:
            n = page * D // 2
            c[..., :n] = torch.randint(0, 256, (pages, H, n), generator=g, device=DEV, dtype=torch.uint8)
            c[..., n:] = torch.randint(123, 128, (pages, H, c.shape[2] - n), generator=g, device=DEV, dtype=torch.uint8)
    return kc, vc


# ------------------------------------------------------------------ append and gather
APPENDS = [  # lengths with the new tokens, new tokens, page, Hk, D, R, interleaved
    ([1], [1], 16, 1, 64, 64, True), ([17, 16, 1, 300], [1, 1, 1, 1], 16, 8, 128, 128, False),
    ([40, 33, 7], [40, 0, 5], 32, 5, 128, 64, False), ([100, 1, 64, 257], [37, 1, 64, 200], 64, 3, 64, 64, True),
    ([500, 20], [130, 20], 256, 4, 128, 128, True), ([90, 31], [50, 31], 128, 2, 64, 16, False),
    ([33, 5, 700], [33, 5, 650], 16, 2, 128, 22, True), ([9] * 70, [9] * 70, 16, 1, 64, 32, False), ([64, 80], [3, 3], 16, 13, 128, 0, True),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{len(c[0])}x{max(c[0])}-" + "-".join(str(x) for x in c[2:]))
def test_append_and_gather(case, dt, bits):
    lens, new, page, Hk, D, R, inter = case
    dtype = DT[dt]
    table, pages = table_for(lens, page, seed=len(lens))
    kc, vc = filled(pages, page, Hk, D, dtype, bits)
    old = [c.clone() for c in (kc, vc)]
    g = torch.Generator(device=DEV).manual_seed(page)
    T = sum(new)
    k, v = (torch.randn(T, Hk, D, generator=g, device=DEV).to(dtype) for _ in "kv")
    k[..., ::17] *= 8
    freqs = prism_amd.rotary_frequencies(R)[0] if R else None
    kw = dict(freqs=freqs, interleaved=inter, amplitude=1.25 if R else 1.0)
    prism_amd.append_paged(k, v, kc, vc, table, ints(lens), cu_seqlens=cu(new), **kw)
    # the definition, written into copies
    who, at = places_of(lens, new)
    where, place = table[who, at // page].long(), at % page
    kr = turned(k, at, freqs, inter, 1.25, dtype) if R else k
    want = [of_cache(c, D) for c in old]
    for w, x in zip(want, (kr, v)):
        w[where, :, place] = x.double() if bits == 16 else levels_of(x)
    for c, w in zip((kc, vc), want):
        assert torch.equal(of_cache(c, D), w)  # (and every other place as it was)
    if len(set(new)) == 1:  # the same without bounds
        again = [c.clone() for c in old]
        prism_amd.append_paged(k, v, *again, table, ints(lens), **kw)
        assert torch.equal(again[0], kc) and torch.equal(again[1], vc)
    # layouts: parts of a projection, [H, T, D] in memory, rows that are not 16-byte aligned
    wide = torch.randn(T, 3 * Hk, D, device=DEV).to(dtype)
    wide[:, Hk:2 * Hk] = v
    odd = torch.empty(T, Hk, D + 1, dtype=dtype, device=DEV)[..., 1:]
    odd.copy_(k)
    for kk, vv in ((k.transpose(0, 1).contiguous().transpose(0, 1), wide[:, Hk:2 * Hk]), (odd, v)):
        again = [c.clone() for c in old]
        prism_amd.append_paged(kk, vv, *again, table, ints(lens), cu_seqlens=cu(new), **kw)
        assert torch.equal(again[0], kc) and torch.equal(again[1], vc)
    # read back
    for out in ((torch.bfloat16, torch.float16) if bits == 4 else (dtype,)):
        gk, gv = prism_amd.gather_paged(kc, vc, table, cu(lens), sum(lens) + 5, head_dim=D, dtype=out)
        who, at = places_of(lens, lens)
        for got, w in zip((gk, gv), want):
            rows = w[table[who, at // page].long(), :, at % page]
            assert got.dtype is out and torch.equal(got[:sum(lens)].double(), rows.to(out).double())
            assert not got[sum(lens):].any()


def test_four_bits_at_borders():
    """Every border between two codes, its neighbours on both sides, signs, zeros, the
    largest and the smallest scales; blocks that hold a NaN or an infinity."""
    for dtype in (torch.bfloat16, torch.float16):
        grid = torch.tensor(LEVELS, dtype=torch.float64)
        mids = (grid[1:] + grid[:-1]) / 2
        base = torch.cat([grid, mids]).repeat(3)
        step = torch.finfo(dtype).eps
        base = (base * torch.tensor([1, 1 + step, 1 - step / 2], dtype=torch.float64).repeat_interleave(15)).clamp(max=6)
        rows = []
        exps = [-8, 0, 5, 100, -100, -124] if dtype == torch.bfloat16 else [-8, 0, 5, 11, -10]
        for e in exps:
            for first in (6.0, 4.5, 3.0 * (1 + step), 3.0):  # (the largest of the block, which sets the scale)
                for part in base.split(31):
                    block = torch.zeros(32, dtype=torch.float64)
                    block[0] = first
                    block[1:1 + len(part)] = part.clamp(max=first) * torch.where(torch.arange(len(part)) % 3 == 0, -1.0, 1.0)
                    rows.append(block * 2.0 ** e)
        rows += [torch.zeros(32, dtype=torch.float64), -torch.zeros(32, dtype=torch.float64)]
        rows.append(torch.full((32,), float(torch.finfo(dtype).smallest_normal), dtype=torch.float64))
        for bad in (math.nan, math.inf, -math.inf):
            block = torch.arange(32, dtype=torch.float64)
            block[7] = bad
            rows.append(block)
        while len(rows) % 2:
            rows.append(torch.ones(32, dtype=torch.float64))
        x = torch.stack(rows).view(-1, 1, 64).to(dtype).to(DEV)
        T = len(x)
        table, pages = table_for([T], 16)
        kc, vc = prism_amd.paged_cache(pages, 16, 1, 64, dtype=dtype, bits=4)
        prism_amd.append_paged(x, x.flip(0), kc, vc, table, ints([T]))
        gk, gv = prism_amd.gather_paged(kc, vc, table, cu([T]), T, head_dim=64)
        want = levels_of(x)
        assert torch.equal(gk.double().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
        assert torch.equal(gv.double().nan_to_num(nan=12345.0), want.flip(0).nan_to_num(nan=12345.0))
        assert torch.isnan(want).any() and want[torch.isfinite(want)].abs().max() >= 6


def test_four_bits_beyond_the_types_largest():
    """The largest level of a type's largest values may lie beyond them: read as infinite, and
    the value below the border is not."""
    for dtype, border, below in ((torch.float16, 57344.0, 49152.0), (torch.bfloat16, 7 * 2.0 ** 125, 6 * 2.0 ** 125)):
        x = torch.zeros(2, 1, 64, dtype=dtype, device=DEV)
        x[0, 0, 3], x[0, 0, 40], x[1, 0, 9] = border, -border, border * (1 - torch.finfo(dtype).eps)
        kc, vc = prism_amd.paged_cache(1, 16, 1, 64, dtype=dtype, bits=4)
        prism_amd.append_paged(x, -x, kc, vc, ints([[0]]), ints([2]))
        gk, gv = prism_amd.gather_paged(kc, vc, ints([[0]]), cu([2]), 2, head_dim=64, dtype=dtype)
        for got, sign in ((gk, 1.0), (gv, -1.0)):
            want = torch.zeros_like(x)
            want[0, 0, 3], want[0, 0, 40], want[1, 0, 9] = sign * math.inf, -sign * math.inf, sign * below
            assert torch.equal(got, want)


def test_caches_that_share_places_are_refused():
    k = torch.randn(2, 4, 64, device=DEV).bfloat16()
    kc, vc = prism_amd.paged_cache(3, 16, 4, 64)
    for kk, vv in ((kc[:, :1].expand_as(kc), vc), (kc, vc[:1].expand_as(vc))):
        with pytest.raises(ValueError, match="share memory"):
            prism_amd.append_paged(k, k, kk, vv, ints([[0], [1]]), ints([1, 1]))
    assert not kc.any() and not vc.any()
    # (to read, they may)
    prism_amd.append_paged(k[:, :1], k[:, :1], *prism_amd.paged_cache(3, 16, 1, 64), ints([[0], [1]]), ints([1, 1]))
    one = [c[:, :1].expand_as(c) for c in (kc, vc)]
    kc[:, :1].normal_()
    vc[:, :1].normal_()
    check(k, *one, ints([[0], [1]]), [9, 16], page=16)


def test_places_that_are_none():
    """Tokens before the table or beyond it, pages that are none, rows of no sequence:
    not stored, and nothing else is changed."""
    page, Hk, D = 16, 2, 64
    table = ints([[2, -1, 5], [7, 99, 1], [0, 3, -7], [4, 6, 8]])
    lens, new = [40, 40, 3, 60], [40, 30, 9, 20]
    for bits in (16, 4):
        kc, vc = filled(9, page, Hk, D, torch.bfloat16, bits)
        before = [of_cache(c, D).clone() for c in (kc, vc)]
        k, v = (torch.randn(sum(new) + 11, Hk, D, device=DEV).bfloat16() for _ in "kv")
        prism_amd.append_paged(k, v, kc, vc, table, ints(lens), cu_seqlens=cu(new) + 4)
        for c, w, x in zip((kc, vc), before, (k, v)):
            row = 4
            for b, (L, n) in enumerate(zip(lens, new)):
                for i in range(n):
                    p = L - n + i
                    if p >= 0 and p // page < 3 and 0 <= int(table[b, p // page]) < 9:
                        w[int(table[b, p // page]), :, p % page] = x[row].double() if bits == 16 else levels_of(x[row])
                    row += 1
            assert torch.equal(of_cache(c, D), w)
        gk, _ = prism_amd.gather_paged(kc, vc, table, cu([48, 48, 70, 0]), 170, head_dim=D)
        held = of_cache(kc, D)
        for b, first, n in ((0, 0, 48), (1, 48, 48), (2, 96, 70)):
            for p in range(n):
                id = int(table[b, p // page]) if p // page < 3 else -1
                want = held[id, :, p % page] if 0 <= id < 9 else torch.zeros(Hk, D, dtype=torch.float64, device=DEV)
                assert torch.equal(gk[first + p].double(), want)
        assert not gk[166:].any()


def test_positions_of_their_own():
    for bits in (16, 4):
        lens = [20, 33]
        T, Hk, D, page = sum(lens), 2, 128, 16
        table, pages = table_for(lens, page)
        k, v = (torch.randn(T, Hk, D, device=DEV).bfloat16() for _ in "kv")
        who, at = places_of(lens, lens)
        where, place = table[who, at // page].long(), at % page
        pos = torch.randint(0, 300000, (T,), device=DEV)
        freqs, amp = prism_amd.rotary_frequencies(128, scaling="yarn", factor=8, original_length=8192)
        grid = torch.randint(0, 90, (T, 3), device=DEV, dtype=torch.int32)
        gf, _ = prism_amd.rotary_frequencies(128, sections=(44, 42, 42))
        for kw, want in ((dict(freqs=freqs, positions=pos, amplitude=amp, interleaved=False), turned(k, pos, freqs, False, amp, k.dtype)),
                         (dict(freqs=freqs, positions=pos[::2].repeat_interleave(2)[:T].int()),
                          turned(k, pos[::2].repeat_interleave(2)[:T], freqs, True, 1.0, k.dtype)),
                         (dict(freqs=gf, positions=grid, sections=(44, 42, 42)), turned(k, grid, gf, True, 1.0, k.dtype, [22, 21, 21]))):
            kc, vc = prism_amd.paged_cache(pages, page, Hk, D, bits=bits)
            prism_amd.append_paged(k, v, kc, vc, table, ints(lens), cu_seqlens=cu(lens), **kw)
            got = of_cache(kc, D)[where, :, place]
            assert torch.equal(got, want.double() if bits == 16 else levels_of(want))


# ------------------------------------------------------------------ attention
def check(q, kc, vc, table, lens, *, page, sm_scale=None):
    T, Hq, D = q.shape
    Hk, B = kc.shape[1], len(lens)
    n, G = T // B, Hq // Hk
    o, lse = prism_amd.flash_attn_paged(q, kc, vc, table, ints(lens), sm_scale=sm_scale, return_lse=True)
    assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (Hq, T)
    scale = D ** -0.5 if sm_scale is None else sm_scale
    four, half = kc.dtype is torch.uint8, q.dtype == torch.float16
    K, V = of_cache(kc, D), of_cache(vc, D)
    u = torch.finfo(q.dtype).eps / 2
    up = 2.0 ** -8 if four else u
    worst = 0.0
    for b, L in enumerate(lens):
        L = min(max(L, 0), table.shape[1] * page)
        at = torch.arange(L, device=DEV)
        ids = table[b, at // page].long()
        there = (ids >= 0) & (ids < kc.shape[0])
        k, v = (c[ids.clamp(0, kc.shape[0] - 1), :, at % page].masked_fill(~there[:, None, None], 0) for c in (K, V))
        rows = slice(b * n, b * n + n)
        qb = q[rows].double().view(n, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * n, D)
        mask = (at <= (L - n + torch.arange(n, device=DEV)).repeat(G)[:, None]) & there
        kt = k.permute(1, 2, 0).contiguous()
        x = (qb @ kt * scale).masked_fill(~mask, -math.inf)
        want_lse = torch.logsumexp(x, -1) if L else torch.full((Hk, G * n), -math.inf, dtype=torch.float64, device=DEV)
        P = torch.exp(x - want_lse.nan_to_num(neginf=0.0)[..., None])
        vt = v.permute(1, 0, 2).contiguous()
        want = P @ vt
        count = mask.sum(-1).double()[None, :, None]
        e = torch.zeros_like(want_lse)[..., None]
        if L:
            e = (qb.abs() @ kt.abs() * scale).masked_fill(~mask, 0).amax(-1, keepdim=True) * (D + 2) * 2.0 ** -24
            if four and half:
                e = e + D * 2.0 ** -25 * qb.abs().amax(-1, keepdim=True) * scale
        tol = (P @ vt.abs()) * (up * 1.001 + 2 * e + count * 2.0 ** -24) + u * want.abs() + torch.finfo(q.dtype).smallest_normal * u
        if half and not four and L:
            tol = tol + count * 2.0 ** -25 * vt.abs().amax(1, keepdim=True)
        back = lambda t: t.view(Hk, G, n, -1).permute(2, 0, 1, 3).reshape(n, Hq, -1)  # noqa: E731
        worst = max(worst, ((o[rows].double() - back(want)).abs() / back(tol)).nan_to_num(math.inf).max().item())
        none = ~mask.any(-1).view(G, n)[0]
        assert (o[rows][none] == 0).all() and (lse[:, rows][:, none] == -math.inf).all()
        wl = want_lse.view(Hq, n)
        ltol = e.view(Hq, n) + (count[0, :, 0].view(G, n)[0] + 8) * 2.0 ** -24 + wl.abs() * 2.0 ** -22 + 2.0 ** -21
        assert ((lse[:, rows].double() - wl).abs() <= ltol)[:, ~none].all()
    assert worst <= 1, f"{worst:.3f} of the bound"
    return o, lse


TOKENS = [  # lengths, new tokens of each, Hq, Hk, D, page
    ([1], 1, 1, 1, 64, 16), ([17, 1, 33], 1, 4, 4, 128, 16), ([1000, 37, 512], 1, 32, 8, 128, 16), ([5000], 1, 8, 1, 64, 32),
    ([700, 64, 65], 5, 6, 3, 128, 64), ([2, 3, 300], 3, 4, 2, 64, 16), ([9001, 12], 2, 64, 2, 64, 128), ([300] * 8, 1, 5, 5, 128, 256),
    ([20000, 0, 2600], 1, 16, 2, 128, 16), ([450, 449], 13, 3, 1, 128, 32), ([64] * 5, 4, 8, 2, 128, 64), ([3000, 70], 1, 28, 4, 128, 16),
    ([100, 2100] * 20, 1, 8, 4, 64, 32), ([130, 7], 40, 8, 8, 64, 16), ([40000], 1, 2, 1, 128, 16), ([1500], 1, 40, 1, 64, 16),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", TOKENS, ids=lambda c: f"{len(c[0])}x{max(c[0])}-" + "-".join(str(x) for x in c[1:]))
def test_tokens(case, dt, bits):
    lens, n, Hq, Hk, D, page = case
    table, pages = table_for(lens, page, seed=n)
    kc, vc = filled(pages, page, Hk, D, DT[dt], bits, seed=len(lens))
    g = torch.Generator(device=DEV).manual_seed(n)
    q = torch.randn(len(lens) * n, Hq, D, generator=g, device=DEV).to(DT[dt])
    a = check(q, kc, vc, table, lens, page=page)
    b = check(q.transpose(0, 1).contiguous().transpose(0, 1), kc, vc, table, lens, page=page)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [16, 4])
def test_tables(bits):
    """Pages that are none in the middle and at the end, lengths beyond the table, below 0,
    a table far wider than the lengths (and not contiguous)."""
    page, D = 16, 128
    lens = [100, 3000, 900, -4, 40]
    table, pages = table_for([100, 2000, 900, 0, 48], page, wide=125)
    table[0, 2] = -1
    table[1, 5:60] = pages + 3
    table[2, :50] = -1
    table[4, 0] = -2
    kc, vc = filled(pages, page, 4, D, torch.bfloat16, bits)
    q = torch.randn(10, 8, D, device=DEV).bfloat16()
    a = check(q, kc, vc, table, lens, page=page, sm_scale=0.3)
    wide = torch.full((5, 4000), 1, dtype=torch.int32, device=DEV)
    wide[:, ::2][:, :125] = table
    wide[:, 250:] = -1
    b = check(q, kc, vc, wide[:, ::2], [100, 2000, 900, -4, 40], page=page, sm_scale=0.3)
    for x, y in zip(a, b):  # (cut otherwise: sums in another order)
        assert torch.allclose(x.float().nan_to_num(neginf=-99.0), y.float().nan_to_num(neginf=-99.0), rtol=2 ** -7, atol=2 ** -8)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("L", [50, 1030])
def test_unused_places_may_hold_anything(bits, L):
    page, D = 32, 64
    for dt in (torch.bfloat16, torch.float16):
        table, pages = table_for([L, L - 13], page)
        kc, vc = filled(pages, page, 2, D, dt, bits)
        q = torch.randn(6, 8, D, device=DEV).to(dt)
        want = check(q, kc, vc, table, [L, L - 13], page=page)
        for b, n in enumerate((L, L - 13)):
            last, used = int(table[b, (n - 1) // page]), (n - 1) % page + 1
            for c in (kc, vc):
                if bits == 16:
                    c[last, :, used:] = float("nan")
                else:
                    c[last, :, page * D // 2 + used * (D // 32):] = 255
        got = prism_amd.flash_attn_paged(q, kc, vc, table, ints([L, L - 13]), return_lse=True)
        assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("L", [90, 2000])
def test_not_finite_reaches_who_sees_it(bits, L):
    page, D, n = 16, 64, 4
    for dt in (torch.bfloat16, torch.float16):
        table, pages = table_for([L, 70], page)
        kc, vc = filled(pages, page, 2, D, dt, bits)
        q = torch.randn(2 * n, 4, D, device=DEV).to(dt)
        want, _ = check(q, kc, vc, table, [L, 70], page=page)
        for place in (L - 2, 3):
            id, at = int(table[0, place // page]), place % page
            for c, bad in ((kc, "nan"), (vc, "nan"), (vc, "inf")):
                old = c.clone()
                if bits == 16:
                    c[id, 1, at, 5] = float(bad)
                else:
                    c[id, 1, page * D // 2 + at * (D // 32)] = 255  # (its first 32 channels)
                o = prism_amd.flash_attn_paged(q, kc, vc, table, ints([L, 70]))
                c.copy_(old)
                hit = torch.zeros(2 * n, 4, dtype=torch.bool, device=DEV)
                hit[max(0, place - (L - n)):n, 2:] = True
                assert torch.isfinite(o[~hit]).all() and not torch.isfinite(o[..., 5][hit]).any()
                assert torch.allclose(o[~hit].float(), want[~hit].float(), rtol=2 ** -6, atol=2 ** -7)


def test_caches_in_larger_tensors():
    """Views of a pool that holds all layers, and of one laid out by place."""
    page, H, D, lens = 16, 4, 128, [70, 33]
    table, pages = table_for(lens, page)
    k, v = (torch.randn(sum(lens), H, D, device=DEV).bfloat16() for _ in "kv")
    q = torch.randn(2, 8, D, device=DEV).bfloat16()
    freqs, _ = prism_amd.rotary_frequencies(D)
    want = None
    for kind in ("own", "layers", "places"):
        if kind == "layers":
            pool = torch.zeros(pages, 2, 3, H, page, D, device=DEV, dtype=torch.bfloat16)
            kc, vc = pool[:, 0, 1], pool[:, 1, 1]
        elif kind == "places":
            pool = torch.zeros(2, pages, page, H, D, device=DEV, dtype=torch.bfloat16)
            kc, vc = pool[0].transpose(1, 2), pool[1].transpose(1, 2)
        else:
            kc, vc = prism_amd.paged_cache(pages, page, H, D)
        prism_amd.append_paged(k, v, kc, vc, table, ints(lens), cu_seqlens=cu(lens), freqs=freqs)
        got = [prism_amd.flash_attn_paged(q, kc, vc, table, ints(lens)), *prism_amd.gather_paged(kc, vc, table, cu(lens), sum(lens))]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    pool = torch.zeros(pages, 2, 3, H, page * (D // 2 + D // 32), device=DEV, dtype=torch.uint8)
    own = prism_amd.paged_cache(pages, page, H, D, bits=4)
    for kc, vc in ((pool[:, 0, 1], pool[:, 1, 1]), own):
        prism_amd.append_paged(k, v, kc, vc, table, ints(lens), cu_seqlens=cu(lens), freqs=freqs)
    assert torch.equal(pool[:, 0, 1], own[0]) and torch.equal(pool[:, 1, 1], own[1]) and not pool[:, :, 0].any()
    assert torch.equal(prism_amd.flash_attn_paged(q, pool[:, 0, 1], pool[:, 1, 1], table, ints(lens)),
                       prism_amd.flash_attn_paged(q, *own, table, ints(lens)))


def test_nothing_to_do():
    kc, vc = prism_amd.paged_cache(2, 16, 2, 64)
    table = torch.full((3, 1), -1, dtype=torch.int32, device=DEV)
    none = torch.empty(0, 2, 64, device=DEV, dtype=torch.bfloat16)
    prism_amd.append_paged(none, none, kc, vc, table, ints([0, 0, 0]), cu_seqlens=ints([0, 0, 0, 0]))
    assert prism_amd.flash_attn_paged(torch.empty(0, 4, 64, device=DEV, dtype=torch.bfloat16), kc, vc, table, ints([0, 0, 0])).shape == (0, 4, 64)
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    o, lse = prism_amd.flash_attn_paged(q, kc, vc, table, ints([0, 5, -1]), return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    k, v = prism_amd.gather_paged(kc, vc, table[:0], ints([0]), 3)
    assert k.shape == (3, 2, 64) and not k.any() and not v.any()
