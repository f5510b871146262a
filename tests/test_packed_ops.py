"""Argument checks of the heads' norms, packed attention and the paged cache, on the
CPU (no kernel runs)."""
import ctypes

import pytest
import torch

import prism_amd
from prism_amd import _lib


def _heads():
    q, k = torch.randn(2, 4, 5, 16), torch.randn(2, 2, 5, 16)
    f, _ = prism_amd.rotary_frequencies(16, device="cpu")
    return q, k, torch.ones(16), f, torch.arange(5)


def test_head_norm_refusals():
    q, k, w, f, at = _heads()
    call = prism_amd.qk_norm_rotary
    with pytest.raises(ValueError, match="GPU"):
        call(q, k, w, w, f, at)
    with pytest.raises(ValueError, match="B, H, S, D"):
        call(q[0], k, w, w, f, at)
    with pytest.raises(ValueError, match="k "):
        call(q, k[:, :, :4], w, w, f, at)
    with pytest.raises(ValueError, match="q_weight"):
        call(q, k, w[:8], w, f, at)
    with pytest.raises(TypeError, match="k_weight"):
        call(q, k, w, w.half(), f, at)
    with pytest.raises(TypeError, match="one dtype"):
        call(q.half(), k.half(), w, w.half(), f, at)
    with pytest.raises(ValueError, match="without k"):
        call(q, None, w, w, f, at)
    with pytest.raises(ValueError, match="eps"):
        call(q, k, w, w, f, at, eps=-1.0)
    with pytest.raises(TypeError, match="float64"):
        call(q, k, w, w, f.float(), at)
    with pytest.raises(ValueError, match="fit"):
        call(q[..., :14], k[..., :14], None, None, f, at)
    with pytest.raises(ValueError, match="sections"):
        call(q, k, w, w, f, at, sections=(8, 6))
    with pytest.raises(ValueError, match="freqs"):
        call(q, k, w, w, f.requires_grad_(True), at)


def test_head_norm_capi_refusals():
    lib = _lib.load()
    one = ctypes.c_void_p(16)
    st, ps, ends = (ctypes.c_int64 * 18)(), (ctypes.c_int64 * 3)(), (ctypes.c_int32 * 4)(8)

    def fwd(dtype=1, wd=0, Hq=2, D=16, R=16, eps=1e-6, axes=1, q=one):
        return lib.prism_qk_norm_rotary(q, one, dtype, 1, 4, Hq, 1, D, R, st, one, one, wd, eps, one, one, 0, ps, axes, ends,
                                        1, 1.0, one, one, None)

    def bwd(partial=one, dy=one, R=16):
        return lib.prism_qk_norm_rotary_bwd(dy, one, one, one, 1, 1, 4, 2, 1, 16, R, st, one, one, 0, 1e-6, one, one, 0, ps, 1,
                                            ends, 1, 1.0, one, one, partial, one, one, None)

    assert [fwd(dtype=3), fwd(wd=2), fwd(Hq=1024), fwd(D=257), fwd(R=15), fwd(R=18), fwd(R=14), fwd(eps=-1.0), fwd(axes=5),
            fwd(q=None)] == [1] * 10
    assert [bwd(partial=None), bwd(dy=None), bwd(R=14)] == [1] * 3


def test_packed_refusals():
    q, k = torch.randn(9, 4, 64).bfloat16(), torch.randn(9, 2, 64).bfloat16()
    b = torch.tensor([0, 4, 9], dtype=torch.int32)
    call = prism_amd.flash_attn_packed
    with pytest.raises(ValueError, match="GPU"):
        call(q, k, k, b)
    with pytest.raises(ValueError, match="Tq, Hq, D"):
        call(q[None], k, k, b)
    with pytest.raises(ValueError, match="Tq, Hq, D"):
        call(q, k, k[:8], b)
    with pytest.raises(ValueError, match="head_dim"):
        call(q[..., :32], k[..., :32], k[..., :32], b)
    with pytest.raises(ValueError, match="evenly"):
        call(q[:, :3], k, k, b)
    with pytest.raises(ValueError, match="evenly"):
        call(q, k[:, :0], k[:, :0], b)
    with pytest.raises(TypeError, match="bfloat16"):
        call(q.float(), k.float(), k.float(), b)
    with pytest.raises(TypeError, match="bfloat16"):
        call(q, k, k.half(), b)
    with pytest.raises(ValueError, match="cu_seqlens_k"):
        call(q[:5], k, k, b)
    with pytest.raises(ValueError, match="cu_seqlens must"):
        call(q, k, k, b.long())
    with pytest.raises(ValueError, match="cu_seqlens must"):
        call(q, k, k, b[:0])
    with pytest.raises(ValueError, match="cu_seqlens_k must"):
        call(q, k, k, b, cu_seqlens_k=b[:2])
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="sm_scale"):
            call(q, k, k, b, sm_scale=bad)


def test_packed_capi_refusals():
    lib = _lib.load()
    one = ctypes.c_void_p(16)
    st = (ctypes.c_int64 * 16)(*[64] * 16)
    odd = (ctypes.c_int64 * 16)(*[63] * 16)
    far = (ctypes.c_int64 * 16)(*[64, 1 << 24] * 8)

    def fwd(dtype=1, B=1, Hq=4, Hk=2, T=9, D=64, s=st, scale=0.1, q=one, cu=one, plan=one, part=one):
        return lib.prism_packed_fwd(q, one, one, dtype, B, Hq, Hk, T, T, D, s, cu, cu, 1, scale, one, None, None, plan, part, None)

    def bwd(T=9, s=st, rest=one, rows=one, plan=one, part=one):
        return lib.prism_packed_bwd(one, one, one, one, one, rest, one, 1, 1, 4, 2, T, T, 64, s, one, one, 1, 0.1, one, one, one,
                                    rows, plan, part, None)

    assert [fwd(dtype=0), fwd(B=-1), fwd(Hq=3), fwd(T=-1), fwd(T=1 << 29), fwd(D=80), fwd(s=odd), fwd(s=far), fwd(scale=0.0),
            fwd(q=None), fwd(cu=None), fwd(q=ctypes.c_void_p(8)), fwd(T=5000, plan=None), fwd(T=5000, part=None)] == [1] * 14
    assert [bwd(s=odd), bwd(rest=None), bwd(rows=None), bwd(T=5000, plan=None), bwd(T=5000, part=None)] == [1] * 5
    ints, floats = ctypes.c_int64(0), ctypes.c_int64(0)
    for B, T in ((1, 10), (7, 301), (3, 16001), (600, 5000), (8, 1 << 20)):
        assert lib.prism_packed_fwd_plan(B, 32, 8, T, T, 128, ctypes.byref(ints), ctypes.byref(floats)) == 0
        # entries of eight ints for every block and part, the parts' sums in 160 MB at most
        assert 0 <= ints.value <= 8 * (2 + T * 4 // 128 + B + 1024) and 0 <= floats.value * 4 <= 160 << 20
        assert lib.prism_packed_bwd_plan(B, 32, 8, T, T, 128, ctypes.byref(ints), ctypes.byref(floats)) == 0
        assert 0 <= floats.value * 4 <= 320 << 20
    assert lib.prism_packed_fwd_plan(1, 3, 2, 10, 10, 128, ctypes.byref(ints), ctypes.byref(floats)) == 1


def _paged(bits=16, D=64, page=16, pages=4, heads=2):
    kc, vc = prism_amd.paged_cache(pages, page, heads, D, bits=bits, device="cpu")
    table = torch.tensor([[0, 1], [2, -1]], dtype=torch.int32)
    return kc, vc, table, torch.tensor([17, 4], dtype=torch.int32)


def test_paged_cache_shapes():
    kc, vc = prism_amd.paged_cache(3, 32, 5, 128, dtype=torch.float16, device="cpu")
    assert kc.shape == vc.shape == (3, 5, 32, 128) and kc.dtype is torch.float16 and not kc.any()
    kc, vc = prism_amd.paged_cache(3, 32, 5, 128, bits=4, device="cpu")
    assert kc.shape == vc.shape == (3, 5, 32 * 68) and kc.dtype is torch.uint8
    for bad in (dict(page_size=24), dict(page_size=8), dict(head_dim=96), dict(pages=0), dict(heads=0), dict(bits=8)):
        with pytest.raises(ValueError):
            prism_amd.paged_cache(**{**dict(pages=3, page_size=32, heads=5, head_dim=128, device="cpu"), **bad})
    with pytest.raises(TypeError):
        prism_amd.paged_cache(3, 32, 5, 128, dtype=torch.float32, device="cpu")


@pytest.mark.parametrize("bits", [16, 4])
def test_append_refusals(bits):
    kc, vc, table, lens = _paged(bits)
    k = torch.randn(2, 2, 64).bfloat16()
    f, _ = prism_amd.rotary_frequencies(64, device="cpu")
    call = prism_amd.append_paged
    with pytest.raises(ValueError, match="GPU"):
        call(k, k, kc, vc, table, lens)
    with pytest.raises(ValueError, match="T, Hk, D"):
        call(k, k[:1], kc, vc, table, lens)
    with pytest.raises(TypeError, match="bfloat16"):
        call(k.float(), k.float(), kc, vc, table, lens)
    with pytest.raises(TypeError, match="bfloat16"):
        call(k, k.half(), kc, vc, table, lens)
    with pytest.raises(ValueError, match="key heads"):
        call(k[:, :1], k[:, :1], kc, vc, table, lens)
    with pytest.raises(ValueError, match="caches must"):
        call(k, k, kc, vc[:3], table, lens)
    with pytest.raises(ValueError, match="caches must" if bits == 16 else "page size"):
        call(torch.cat([k, k], -1), torch.cat([k, k], -1), kc, vc, table, lens)
    with pytest.raises(ValueError, match="head_dim"):
        call(k[..., :32], k[..., :32], kc, vc, table, lens)
    with pytest.raises(TypeError, match="caches must"):
        call(k, k, kc.float(), vc.float(), table, lens)
    with pytest.raises(ValueError, match="page size"):
        call(k, k, kc[:, :, :8 if bits == 16 else 8 * 34], vc[:, :, :8 if bits == 16 else 8 * 34], table, lens)
    with pytest.raises(ValueError, match="page_table"):
        call(k, k, kc, vc, table.long(), lens)
    with pytest.raises(ValueError, match="page_table"):
        call(k, k, kc, vc, table[:, :0], lens)
    with pytest.raises(ValueError, match="kv_lens"):
        call(k, k, kc, vc, table, lens[:1])
    with pytest.raises(ValueError, match="kv_lens"):
        call(k, k, kc, vc, table, lens.long())
    with pytest.raises(ValueError, match="cu_seqlens"):
        call(k, k, kc, vc, table, lens, cu_seqlens=lens)
    with pytest.raises(ValueError, match="share out"):
        call(k[:1], k[:1], kc, vc, table, lens)
    with pytest.raises(ValueError, match="gradient"):
        call(k.clone().requires_grad_(True), k, kc, vc, table, lens)
    with pytest.raises(TypeError, match="float64"):
        call(k, k, kc, vc, table, lens, freqs=f.float())
    with pytest.raises(ValueError, match="fit"):
        call(k, k, kc, vc, table, lens, freqs=torch.cat([f, f]))
    with pytest.raises(ValueError, match="multiple of 16"):
        call(k, k, kc, vc, table, lens, freqs=f[:12], interleaved=False)
    with pytest.raises(ValueError, match="go with freqs"):
        call(k, k, kc, vc, table, lens, positions=lens)
    with pytest.raises(ValueError, match="sections need"):
        call(k, k, kc, vc, table, lens, freqs=f, sections=(32, 32))
    with pytest.raises(ValueError, match="sections"):
        call(k, k, kc, vc, table, lens, freqs=f, sections=(32, 30), positions=table)
    with pytest.raises(ValueError, match="positions must"):
        call(k, k, kc, vc, table, lens, freqs=f, positions=lens[:1])
    if bits == 16:
        with pytest.raises(TypeError, match="k's dtype"):
            call(k.half(), k.half(), kc, vc, table, lens)


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_refusals(bits):
    kc, vc, table, lens = _paged(bits)
    q = torch.randn(4, 8, 64).bfloat16()
    call = prism_amd.flash_attn_paged
    with pytest.raises(ValueError, match="GPU"):
        call(q, kc, vc, table, lens)
    with pytest.raises(ValueError, match="T, Hq, D"):
        call(q[0], kc, vc, table, lens)
    with pytest.raises(TypeError, match="bfloat16"):
        call(q.float(), kc, vc, table, lens)
    with pytest.raises(ValueError, match="evenly"):
        call(q[:, :5], kc, vc, table, lens)
    with pytest.raises(ValueError, match="evenly"):
        call(q[:, :1], kc, vc, table, lens)
    with pytest.raises(ValueError, match="share out"):
        call(q[:3], kc, vc, table, lens)
    with pytest.raises(ValueError, match="kv_lens"):
        call(q, kc, vc, table, lens[None])
    with pytest.raises(ValueError, match="gradient"):
        call(q.clone().requires_grad_(True), kc, vc, table, lens)
    with pytest.raises(ValueError, match="sm_scale"):
        call(q, kc, vc, table, lens, sm_scale=0.0)
    if bits == 16:
        with pytest.raises(TypeError, match="q's dtype"):
            call(q.half(), kc, vc, table, lens)
    g = prism_amd.gather_paged
    b = torch.tensor([0, 3, 9], dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        g(kc, vc, table, b, 9, head_dim=64)
    with pytest.raises(ValueError, match="cu_seqlens"):
        g(kc, vc, table, b[:2], 9, head_dim=64)
    with pytest.raises(ValueError, match="total"):
        g(kc, vc, table, b, -1, head_dim=64)
    with pytest.raises(TypeError, match="dtype"):
        g(kc, vc, table, b, 9, head_dim=64, dtype=torch.float32)
    if bits == 4:
        with pytest.raises(ValueError, match="head_dim"):
            g(kc, vc, table, b, 9)
    else:
        with pytest.raises(TypeError, match="dtype"):
            g(kc, vc, table, b, 9, dtype=torch.float16)


def test_paged_capi_refusals():
    lib = _lib.load()
    one, off = ctypes.c_void_p(16), ctypes.c_void_p(8)
    st = (ctypes.c_int64 * 4)(64, 64, 64, 64)
    odd = (ctypes.c_int64 * 4)(63, 64, 64, 64)
    cs = (ctypes.c_int64 * 6)(*[64] * 6)
    bad = (ctypes.c_int64 * 6)(*[72] * 5, 60)
    far = (ctypes.c_int64 * 6)(*[64] * 5, 1 << 24)
    ends = (ctypes.c_int32 * 4)(8)
    ps = (ctypes.c_int64 * 2)(1, 1)

    def append(dtype=1, T=4, Hk=2, D=64, s=st, kc=one, bits=16, pages=4, page=16, c=cs, table=one, width=2, lens=one, B=2,
               cu=None, freqs=one, R=64, inter=1, pos=None, axes=1, k=one):
        return lib.prism_paged_append(k, one, dtype, T, Hk, D, s, kc, one, bits, pages, page, c, table, 2, width, lens, B, cu,
                                      freqs, R, inter, pos, 0, ps, axes, ends, 1.0, None)

    assert [append(dtype=0), append(T=-1), append(T=3), append(Hk=0), append(D=80), append(s=odd), append(kc=None), append(kc=off),
            append(bits=8), append(pages=0), append(page=24), append(page=512), append(page=8), append(c=bad), append(c=far),
            append(table=None), append(width=0), append(width=1 << 28), append(lens=None), append(B=-1), append(R=63), append(R=66),
            append(R=24, inter=0), append(pos=one, axes=5), append(pos=one), append(k=None), append(k=off),
            append(bits=4, c=(ctypes.c_int64 * 6)(*[72] * 6))] == [1] * 28

    def gather(dtype=1, bits=4, D=64, T=4, cu=one, k=one, page=16):
        return lib.prism_paged_gather(one, one, dtype, bits, 4, page, cs, one, 2, 2, 2, cu, T, 2, D, k, one, None)

    assert [gather(dtype=0), gather(bits=2), gather(D=32), gather(T=-1), gather(cu=None), gather(k=None), gather(k=off),
            gather(page=17)] == [1] * 8

    def fwd(dtype=1, n=1, Hq=4, Hk=2, s=st, scale=0.1, bits=16, width=2, q=one, lens=one, part=one, B=2):
        return lib.prism_paged_fwd(q, dtype, B, n, Hq, Hk, 64, s, one, one, bits, 4, 16, cs, one, 2, width, lens, scale, one, None,
                                   part, None)

    assert [fwd(dtype=0), fwd(n=-1), fwd(n=1 << 30), fwd(Hq=3), fwd(Hq=1), fwd(s=odd), fwd(scale=0.0), fwd(scale=float("nan")),
            fwd(bits=5), fwd(q=None), fwd(q=off), fwd(lens=None), fwd(width=4000, part=None), fwd(bits=4, width=4000, part=None),
            fwd(part=off)] == [1] * 15
    floats = ctypes.c_int64(0)
    for B, n, places, bits in ((1, 1, 100, 16), (16, 1, 8192, 16), (8, 1, 131072, 4), (1, 3, 1 << 20, 4), (500, 1, 1 << 20, 16)):
        assert lib.prism_paged_plan(B, n, 32, 8, 128, bits, places, ctypes.byref(floats)) == 0
        assert 0 <= floats.value * 4 <= 64 << 20
    assert lib.prism_paged_plan(1, 1, 3, 2, 128, 16, 100, ctypes.byref(floats)) == 1
