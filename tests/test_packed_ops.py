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
