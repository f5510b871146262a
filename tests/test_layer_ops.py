"""Argument checks of the layer's operators and the rotary frequencies, on the
CPU (no kernel runs)."""
import ctypes
import math

import pytest
import torch

import prism_amd
from prism_amd import _lib


def test_norm_refusals():
    x = torch.randn(3, 8)
    w = torch.ones(8)
    with pytest.raises(ValueError, match="GPU"):
        prism_amd.rms_norm(x, w)
    with pytest.raises(ValueError, match="GPU"):
        prism_amd.rms_norm_quant(x, w)
    with pytest.raises(ValueError, match="weight"):
        prism_amd.rms_norm(x, torch.ones(7))
    with pytest.raises(TypeError, match="weight"):
        prism_amd.rms_norm(x, w.double())
    with pytest.raises(TypeError, match="residual"):
        prism_amd.rms_norm(x, w, residual=x.half())
    with pytest.raises(ValueError, match="residual"):
        prism_amd.rms_norm(x, w, residual=x[:2])
    with pytest.raises(ValueError, match="eps"):
        prism_amd.rms_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="last dimension"):
        prism_amd.rms_norm(torch.randn(3, 0))
    with pytest.raises(ValueError, match="gradient"):
        prism_amd.rms_norm_quant(x.requires_grad_(True), w)


def test_norm_capi_refusals():
    lib = _lib.load()
    one = ctypes.c_void_p(16)
    for M, N, dtype, out in ((4, 0, 0, 0), (4, 16385, 0, 0), (-1, 8, 0, 0), (4, 8, 5, 5), (4, 8, 1, 0), (4, 8, 1, 3)):
        # (the last: 8 bits without scales)
        assert lib.prism_rms_norm(one, N, None, 0, None, dtype, dtype, M, N, 1e-6, None, one, out, None, None, None) == 1
    assert lib.prism_rms_norm(one, 8, one, 8, None, 1, 1, 4, 8, 1e-6, None, one, 1, None, None, None) == 1  # h missing
    assert lib.prism_rms_norm_bwd(one, 8, None, 0, one, 8, None, 1, 1, 4, 8, one, one, None, 1, one, None) == 1
    parts = ctypes.c_int(0)
    assert lib.prism_rms_norm_parts(75600, 5120, ctypes.byref(parts)) == 0 and 1 <= parts.value <= 1024
    assert lib.prism_rms_norm_parts(0, 5120, ctypes.byref(parts)) == 1


def test_rotary_refusals():
    q = torch.randn(1, 2, 5, 16)
    f, _ = prism_amd.rotary_frequencies(16, device="cpu")
    at = torch.arange(5)
    with pytest.raises(ValueError, match="GPU"):
        prism_amd.apply_rotary(q, None, f, at)
    with pytest.raises(TypeError, match="float64"):
        prism_amd.apply_rotary(q, None, f.float(), at)
    with pytest.raises(ValueError, match="fit"):
        prism_amd.apply_rotary(q[..., :14], None, f, at)
    with pytest.raises(ValueError, match="k "):
        prism_amd.apply_rotary(q, q[:, :, :4], f, at)
    with pytest.raises(ValueError, match="B, H, S, D"):
        prism_amd.apply_rotary(q[0], None, f, at)
    with pytest.raises(ValueError, match="sections"):
        prism_amd.apply_rotary(q, None, f, at, sections=(8, 6))


def test_rotary_capi_refusals():
    lib = _lib.load()
    one = ctypes.c_void_p(16)
    strides, ps, ends = (ctypes.c_int64 * 12)(), (ctypes.c_int64 * 3)(), (ctypes.c_int32 * 4)(8)
    call = lambda dtype=1, D=16, R=16, axes=1, q=one: lib.prism_rotary(  # noqa: E731
        q, None, dtype, 1, 4, 2, 0, D, R, strides, one, one, 0, ps, axes, ends, 1, 1.0, 0, one, None, None)
    assert [call(dtype=3), call(D=257), call(R=15), call(R=18), call(axes=5), call(axes=0), call(q=None), call(R=14)] == [1] * 8


def test_frequencies():
    f, a = prism_amd.rotary_frequencies(8, device="cpu")
    assert a == 1.0 and torch.allclose(f, torch.tensor([1, 0.1, 0.01, 0.001], dtype=torch.float64))
    f2, _ = prism_amd.rotary_frequencies(128, sections=(44, 42, 42), device="cpu")
    one, _ = prism_amd.rotary_frequencies(42, device="cpu")
    assert f2.shape == (64,) and torch.equal(f2[22:43], one) and torch.equal(f2[43:], one)
    lin, _ = prism_amd.rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(lin, f / 4)
    ntk, _ = prism_amd.rotary_frequencies(8, scaling="ntk", factor=4.0, device="cpu")
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    # yarn: the fastest pairs kept, the slowest divided, amplitude grown
    plain, _ = prism_amd.rotary_frequencies(128, device="cpu")
    yarn, a = prism_amd.rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=8192, device="cpu")
    turns = plain * 8192 / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], plain[turns > 40]) and torch.allclose(yarn[turns < 0.8], plain[turns < 0.8] / 8)
    assert math.isclose(a, 0.1 * math.log(8) + 1) and (yarn <= plain).all() and (yarn >= plain / 8 * (1 - 1e-12)).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, sections=(4, 2)), dict(rotary_dim=8, scaling="x"),
                dict(rotary_dim=8, scaling="yarn", factor=2.0), dict(rotary_dim=8, base=0.5), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=4, sections=(2, 2), scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            prism_amd.rotary_frequencies(device="cpu", **bad)


def test_grid_positions_cpu():
    assert prism_amd.grid_positions((1, 2, 2), device="cpu").tolist() == [[0, 0, 0], [0, 0, 1], [0, 1, 0], [0, 1, 1]]


def test_window_refusals():
    q, k = torch.randn(2, 4, 5, 64).bfloat16(), torch.randn(2, 2, 9, 64).bfloat16()
    call = prism_amd.flash_attn_window
    with pytest.raises(ValueError, match="GPU"):
        call(q, k, k, 3)
    with pytest.raises(ValueError, match="B, H, S, D"):
        call(q[0], k, k, 3)
    with pytest.raises(ValueError, match="mismatch"):
        call(q, k, k[:, :, :8], 3)
    with pytest.raises(ValueError, match="mismatch"):
        call(q, k[:1], k[:1], 3)
    with pytest.raises(ValueError, match="head_dim"):
        call(q[..., :32], k[..., :32], k[..., :32], 3)
    with pytest.raises(ValueError, match="evenly"):
        call(q[:, :3], k, k, 3)
    with pytest.raises(ValueError, match="evenly"):
        call(q, k[:, :0], k[:, :0], 3)
    with pytest.raises(TypeError, match="bfloat16"):
        call(q.float(), k.float(), k.float(), 3)
    with pytest.raises(TypeError, match="bfloat16"):
        call(q, k, k.half(), 3)
    with pytest.raises(ValueError, match="window"):
        call(q, k, k, 0)
    with pytest.raises(ValueError, match="sinks"):
        call(q, k, k, 3, sinks=-1)
    for lens in (torch.ones(2), torch.ones(3, dtype=torch.int32), torch.ones(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="kv_lens"):
            call(q, k, k, 3, kv_lens=lens)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="sm_scale"):
            call(q, k, k, 3, sm_scale=scale)


def test_window_capi_refusals():
    lib = _lib.load()
    one = ctypes.c_void_p(16)

    def fwd(dtype=1, B=1, Hq=4, Hk=2, Sq=5, Sk=9, D=64, window=3, sinks=0, scale=0.1, stride=64, p=one):
        st = (ctypes.c_int64 * 12)(*[stride] * 12)
        return lib.prism_window_fwd(p, one, one, dtype, B, Hq, Hk, Sq, Sk, D, st, window, sinks, 1, None, None, scale, one,
                                    None, None, one, None)

    for bad in (dict(dtype=0), dict(Hk=3), dict(Hk=0), dict(D=32), dict(window=0), dict(sinks=-1), dict(scale=0.0),
                dict(stride=65), dict(stride=1 << 24), dict(stride=-64), dict(p=None), dict(p=ctypes.c_void_p(8)),
                dict(Sq=1 << 30), dict(Sk=1 << 30), dict(B=-1)):
        assert fwd(**bad) == 1, bad
    assert fwd(B=0) == 0
    st = (ctypes.c_int64 * 24)(*[64] * 24)
    token = lambda splits, ws: lib.prism_window_token(  # noqa: E731
        one, one, one, 1, 1, 4, 2, 1, 9, 64, st, 3, 0, 1, None, None, 0.1, one, None, None, splits, ws, ws, None)
    assert [token(0, one), token(257, one), token(2, None)] == [1, 1, 1]
    bwd = lambda lse, rows: lib.prism_window_bwd(  # noqa: E731
        one, one, one, one, one, None, lse, 1, 1, 4, 2, 5, 9, 64, st, 3, 0, 1, None, None, 0.1, one, one, one, rows, None, None)
    assert [bwd(None, one), bwd(one, None)] == [1, 1]


def test_window_plans():
    """Workspaces stay small against the tensors: a bounded number of pieces."""
    lib = _lib.load()
    splits, floats = ctypes.c_int(0), ctypes.c_int64(0)
    for B, Hq, Hk, Sq, Sk, W, sinks in ((8, 32, 8, 1, 32768, 4096, 4), (1, 1, 1, 1, 1 << 28, 1 << 28, 0), (1, 8, 8, 1, 1, 1, 0),
                                        (1, 64, 1, 1, 100000, 100000, 0), (0, 4, 4, 1, 5, 5, 0), (64, 32, 8, 2, 9, 5, 2)):
        assert lib.prism_window_token_plan(B, Hq, Hk, Sq, Sk, W, sinks, 1, ctypes.byref(splits), ctypes.byref(floats)) == 0
        assert 1 <= splits.value <= 256
        assert splits.value == 1 or splits.value * 16 <= Sk
        assert floats.value == (0 if splits.value == 1 else splits.value * 32 * B * Hk * -(-Sq * Hq // Hk // 32))
    # many rows over many keys are the other kernel's
    assert lib.prism_window_token_plan(8, 32, 8, 16, 32768, 4096, 4, 1, ctypes.byref(splits), ctypes.byref(floats)) == 0
    assert splits.value == 0 and floats.value == 0
    for B, Hq, Hk, Sq, Sk, W, sinks in ((1, 5, 5, 14040, 14040, 4680, 1560), (1, 1, 1, 200000, 200000, 64, 4), (1, 1, 1, 1, 1, 1, 0),
                                        (4, 32, 8, 16384, 16384, 1 << 29, 0)):
        assert lib.prism_window_fwd_plan(B, Hq, Hk, Sq, Sk, 128, W, sinks, 1, ctypes.byref(floats)) == 0
        assert 0 <= floats.value <= 2 * 512 * 128 * 130
        for D, lens in ((128, 0), (128, 1), (64, 0), (64, 1)):
            assert lib.prism_window_bwd_plan(B, Hq, Hk, Sq, Sk, D, W, sinks, 1, lens, ctypes.byref(floats)) == 0
            assert 0 <= floats.value <= 3000 * 256 * 128


def test_fake_tensors():
    """Traced without a GPU: shapes, layouts and which outputs carry gradients."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from prism_amd import _torch_ops
    _torch_ops.load()
    bf = torch.bfloat16
    with FakeTensorMode():
        for grad in (False, True):
            def mk(*s):
                return torch.empty(*s, device="cuda", dtype=bf, requires_grad=grad)  # noqa: B023
            x, w = mk(3, 5, 64), mk(64)
            y, h = prism_amd.rms_norm(x, w, residual=x)
            assert y.shape == h.shape == x.shape and y.dtype == bf and y.requires_grad == h.requires_grad == grad
            codes, scales = prism_amd.rms_norm_quant(x.detach(), out_dtype=torch.int8)
            assert codes.dtype == torch.int8 and scales.shape == (3, 5) and scales.dtype == torch.float32
            q, k = mk(2, 9, 4, 64).transpose(1, 2), mk(2, 9, 2, 64).transpose(1, 2)
            freqs = torch.empty(32, device="cuda", dtype=torch.float64)
            a, b = prism_amd.apply_rotary(q, k, freqs, torch.empty(9, device="cuda", dtype=torch.int64))
            assert a.stride() == q.stride() and b.stride() == k.stride() and a.requires_grad == grad
            o, lse = prism_amd.flash_attn_window(a, b, b, 5, return_lse=True)
            assert o.stride() == q.stride() and lse.shape == (2, 4, 9)
            assert o.requires_grad == grad and not lse.requires_grad
            odd = mk(2, 4, 9, 65)[..., 1:]
            assert prism_amd.flash_attn_window(odd, odd, odd, 5).shape == (2, 4, 9, 64)


def test_frequencies_take_no_gradient():
    q, freqs = torch.randn(1, 1, 3, 8), torch.ones(4, dtype=torch.float64, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        prism_amd.apply_rotary(q, None, freqs, torch.arange(3))


def test_window_plans_with_every_key_a_sink():
    """Windows and sinks far beyond any length plan like ones of the length."""
    lib = _lib.load()
    far = 1 << 62

    def plans(window, sinks):
        splits, a, b, c = ctypes.c_int(), ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
        assert lib.prism_window_token_plan(2, 8, 2, 1, 5000, window, sinks, 1, ctypes.byref(splits), ctypes.byref(a)) == 0
        assert lib.prism_window_fwd_plan(2, 8, 2, 900, 5000, 64, window, sinks, 1, ctypes.byref(b)) == 0
        assert lib.prism_window_bwd_plan(2, 8, 2, 900, 5000, 64, window, sinks, 1, 1, ctypes.byref(c)) == 0
        return splits.value, a.value, b.value, c.value

    # few keys: the backward needs nothing of o's rounding
    assert [lib.prism_window_rest(*a) for a in ((5000, 64, 0, 1), (5000, 60, 4, 1), (64, far, far, 0), (5000, 32, 1, 0),
                                                (0, 5, 0, 1))] == [0] * 5
    assert [lib.prism_window_rest(*a) for a in ((5000, 65, 0, 1), (5000, 60, 5, 1), (65, far, 0, 1), (5000, 33, 0, 0),
                                                (5000, 1, far, 1))] == [1] * 5
    assert plans(far, far) == plans(5000, 5000)
    assert plans(100, far) == plans(100, 5000)
