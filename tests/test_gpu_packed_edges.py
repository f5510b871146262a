"""Corners of packed batches and paged caches: blocks of 4 bits that are not finite, amplitudes
that float32 does not hold, operator calls without channels, caches that are one, bounds that overlap
(nothing beside a call's outputs and workspaces is written), infinities in head norms."""
import ctypes
import math

import pytest
import torch

import prism_amd
from prism_amd import _lib
from tests.test_gpu_paged import ints, levels_of, of_cache, places_of, table_for, turned

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, dt=torch.bfloat16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dt)


# ------------------------------------------------------------------ 4 bits
@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_blocks_that_are_not_finite_are_nan(dt, D, n):
    """32 channels of which one is not finite are read as NaN, whatever codes stand beside
    their scale: those channels of every token that sees them are NaN (no infinities, whose
    sign would mean nothing), all else is as it was, parts of long sequences too."""
    Hq, Hk, page = 8, 2, 16
    for L in (40, 1500):
        lens = [L, 30]
        table, pages = table_for(lens, page)
        kc, vc = prism_amd.paged_cache(pages, page, Hk, D, bits=4)
        k, v, q = (randn(*s, dt=dt, seed=i) for i, s in enumerate(((L + 30, Hk, D), (L + 30, Hk, D), (2 * n, Hq, D))))
        bounds = ints([0, L, L + 30])
        want = None
        for place, channel, bad in ((None, 0, 0.0), (L - 2, 5, math.nan), (3, 40, math.inf), (L // 2, D - 1, -math.inf)):
            x = v.clone()
            if place is not None:
                x[place, 1, channel] = bad
            prism_amd.append_paged(k, x, kc, vc, table, ints(lens), cu_seqlens=bounds)
            o = prism_amd.flash_attn_paged(q, kc, vc, table, ints(lens))
            if place is None:
                want = o
                assert torch.isfinite(o).all()
                continue
            hit = torch.zeros(2 * n, Hq, D, dtype=torch.bool, device=DEV)
            hit[max(0, place - (L - n)):n, Hq // Hk:, channel // 32 * 32:channel // 32 * 32 + 32] = True
            assert torch.equal(torch.isnan(o), hit) and torch.equal(o[~hit], want[~hit])


# ------------------------------------------------------------------ appended keys
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("bits", [16, 4])
def test_amplitudes_that_float32_does_not_hold(bits, interleaved):
    """yarn's amplitude at factor 40, 0.1 ln 40 + 1, is 3.2e-8 off in float32: the keys are those
    of the float64 rotation, in float16 and its 4 bits, bit for bit (600,000 of them: some 27
    would fall on another side of a border)."""
    Hk, D, page, dt = 8, 128, 64, torch.float16
    lens = [400, 200]
    T = sum(lens)
    table, pages = table_for(lens, page)
    k = randn(T, Hk, D, dt=dt, seed=3)
    freqs, amplitude = prism_amd.rotary_frequencies(D, scaling="yarn", factor=40, original_length=8192)
    assert abs(amplitude - torch.tensor(amplitude).item()) > 2e-8
    who, at = places_of(lens, lens)
    kc, vc = prism_amd.paged_cache(pages, page, Hk, D, dtype=dt, bits=bits)
    prism_amd.append_paged(k, k, kc, vc, table, ints(lens), cu_seqlens=ints([0, 400, 600]), freqs=freqs, amplitude=amplitude,
                           interleaved=interleaved)
    want = turned(k, at, freqs, interleaved, amplitude, dt)
    got = of_cache(kc, D)[table[who, at // page].long(), :, at % page]
    assert torch.equal(got, want.double() if bits == 16 else levels_of(want))


def test_operators_without_channels_are_refused():
    """Heads of no channels, which the functions of prism_amd refuse, as an error of the
    operators beneath them too."""
    table, lens = ints([[0]]), ints([1])
    for dt in (torch.uint8, torch.bfloat16):
        c = torch.zeros((1, 2, 0) if dt is torch.uint8 else (1, 2, 16, 0), dtype=dt, device=DEV)
        x = torch.zeros(1, 2, 0, dtype=torch.bfloat16, device=DEV)
        with pytest.raises(ValueError):
            torch.ops.prism.paged_append(x, x, c, c.clone(), table, lens, None, None, None, [], True, 1.0)
        with pytest.raises(ValueError):
            torch.ops.prism.paged_fwd(x, c, c, table, lens, 2, 0.125, False)
        with pytest.raises(ValueError):
            torch.ops.prism.paged_gather(c, c, table, ints([0, 1]), 1, 2, 0, False)


@pytest.mark.parametrize("bits", [16, 4])
def test_one_cache_for_keys_and_values_is_refused(bits):
    table, lens = ints([[0, 1]]), ints([20])
    x = randn(20, 2, 64)
    pool = torch.stack([c for c in prism_amd.paged_cache(2, 16, 2, 64, bits=bits)], 1)  # [pages, 2, ..]
    kc, _ = prism_amd.paged_cache(2, 16, 2, 64, bits=bits)
    for a, b in ((kc, kc), (kc, kc.view(kc.shape)), (pool[:, 1], pool[:, 1])):
        with pytest.raises(ValueError, match="share memory"):
            prism_amd.append_paged(x, x, a, b, table, lens)
    assert not kc.any() and not pool.any()
    prism_amd.append_paged(x, x, pool[:, 0], pool[:, 1], table, lens)
    assert torch.equal(pool[:, 0], pool[:, 1]) and pool.any()
    # (to read, one may be both)
    o = prism_amd.flash_attn_paged(x[:1], pool[:, 0], pool[:, 0], table, lens)
    assert torch.equal(o, prism_amd.flash_attn_paged(x[:1], pool[:, 0], pool[:, 1], table, lens))


# ------------------------------------------------------------------ bounds that overlap
class Guarded:
    """Buffers inside larger ones of a value that nothing else has."""

    def __init__(self):
        self.all = []

    def __call__(self, shape, dtype):
        n, pad, mark = math.prod(shape), 4096, 1234567 if dtype is torch.int32 else -19.75
        t = torch.full((n + 2 * pad,), mark, dtype=dtype, device=DEV)
        self.all.append((t, n, pad, mark))
        return t[pad:pad + n].view(shape)

    def intact(self):
        return all((t[:pad] == m).all() and (t[pad + n:] == m).all() for t, n, pad, m in self.all)


@pytest.mark.parametrize("causal", [1, 0])
@pytest.mark.parametrize("B", [5, 61, 700])
def test_bounds_that_overlap_write_nothing_else(B, causal):
    """Outputs and workspaces of exactly the planned sizes: with bounds in any order, and with
    hundreds of sequences that each take all tokens, nothing beside them is written, and the
    lists' counts stay within their room."""
    lib = _lib.load()
    T, Hq, Hk, D = 1500, 4, 2, 64
    g = torch.Generator(device=DEV).manual_seed(B)
    any_ = [torch.randint(-99, T + 99, (B + 1,), generator=g, device=DEV, dtype=torch.int32) for _ in "qk"]
    whole = ints([0 if i % 2 == 0 else T for i in range(B + 1)])
    q, k, do = randn(T, Hq, D, seed=1), randn(T, Hk, D, seed=2), randn(T, Hq, D, seed=3)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    sizes = []
    for plan in (lib.prism_packed_fwd_plan, lib.prism_packed_bwd_plan):
        ints_, floats = ctypes.c_int64(0), ctypes.c_int64(0)
        assert plan(B, Hq, Hk, T, T, D, ctypes.byref(ints_), ctypes.byref(floats)) == 0
        sizes.append((ints_.value, floats.value))
    assert all(n > 0 for n, _ in sizes) and (B == 700 or all(n > 0 for _, n in sizes))  # (lists, and blocks that may be cut)
    st = lambda *ts: (ctypes.c_int64 * (2 * len(ts)))(*[s for t in ts for s in (t.stride(1), t.stride(0))])  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for cq, ck in (any_, any_[::-1], (whole, whole), (whole, any_[0])):
        new, bf, f32, i32 = Guarded(), torch.bfloat16, torch.float32, torch.int32
        o, rest, lse, dq, dk, dv = (new(s, t) for s, t in (((T, Hq, D), bf), ((T, Hq, D), bf), ((Hq, T), f32), ((T, Hq, D), bf),
                                                          ((T, Hk, D), bf), ((T, Hk, D), bf)))
        plans, parts, rows = [new((n,), i32) for n, _ in sizes], [new((n,), f32) for _, n in sizes], new((2 * Hq * T,), f32)
        rest.zero_()  # (rows that an overlap leaves out are read by the backward)
        o.zero_()
        lse.zero_()
        torch.cuda.synchronize()
        assert lib.prism_packed_fwd(ptr(q), ptr(k), ptr(k), 1, B, Hq, Hk, T, T, D, st(q, k, k, o), ptr(cq), ptr(ck), causal, 0.125,
                                    ptr(o), ptr(rest), ptr(lse), ptr(plans[0]), ptr(parts[0]), stream) == 0
        assert lib.prism_packed_bwd(ptr(do), ptr(q), ptr(k), ptr(k), ptr(o), ptr(rest), ptr(lse), 1, B, Hq, Hk, T, T, D,
                                    st(q, k, k, o, do, dq, dk, dv), ptr(cq), ptr(ck), causal, 0.125, ptr(dq), ptr(dk), ptr(dv),
                                    ptr(rows), ptr(plans[1]), ptr(parts[1]), stream) == 0
        torch.cuda.synchronize()
        assert new.intact()
        for plan, (n, _) in zip(plans, sizes):  # (entries and cuts of eight ints behind the first eight)
            entries, cuts, pieces = plan[:3].tolist()
            assert 0 <= entries and 0 <= cuts and 8 * (1 + entries) <= n and 8 * (1 + cuts) <= n and pieces >= 0


# ------------------------------------------------------------------ head norms
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (36, 36), (36, 16)])
def test_infinities_in_a_head(D, R, dt):
    """A NaN fills its head; beside an infinity the inverse root is 0, so that its own channel
    and the one that turns with it (if it turns) are NaN and the head's others 0; squares whose
    sum passes float32's range give 0 alike."""
    q = randn(1, 4, 6, D, dt=dt, seed=1)
    freqs, _ = prism_amd.rotary_frequencies(R)
    at = torch.arange(1, 7, device=DEV)
    for inter in (True, False):
        partner = lambda c: c if c >= R else c ^ 1 if inter else (c + R // 2) % R  # noqa: E731
        x = q.clone()
        x[0, 0, 1, 5], x[0, 1, 2, 9], x[0, 2, 3, D - 1] = math.nan, math.inf, -math.inf
        if dt is not torch.float16:
            x[0, 3, 4, 2] = 3e19
        y = prism_amd.qk_norm_rotary(x, None, None, None, freqs, at, interleaved=inter)
        want = prism_amd.qk_norm_rotary(q, None, None, None, freqs, at, interleaved=inter)
        want[0, 0, 1] = math.nan
        for h, s, c in ((1, 2, 9), (2, 3, D - 1)):
            want[0, h, s] = 0
            want[0, h, s, [c, partner(c)]] = math.nan
        if dt is not torch.float16:
            want[0, 3, 4] = 0
        assert torch.equal(y.nan_to_num(nan=99.0), want.nan_to_num(nan=99.0))
