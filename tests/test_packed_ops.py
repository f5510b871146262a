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
