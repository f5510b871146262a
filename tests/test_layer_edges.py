"""Corners of the layer's operators, on the CPU (no kernel runs)."""
import ctypes
import math

import pytest
import torch

import prism_amd


@pytest.mark.parametrize("dim,factor,length", [(128, 8.0, 65536), (128, 8.0, 131072), (8, 8.0, 8192), (64, 4.0, 8192),
                                               (128, 16.0, 4096), (32, 2.0, 1 << 20)])
def test_yarn_ramp_past_the_last_pair(dim, factor, length):
    """The ramp ends where a pair would turn beta_slow times, past the head's last
    pair too: pairs that turn more often than that are not divided in full."""
    fast, slow, base = 32.0, 1.0, 10000.0
    f, _ = prism_amd.rotary_frequencies(dim, base=base, scaling="yarn", factor=factor, original_length=length, device="cpu")
    where = lambda n: dim * math.log(length / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(where(fast)), 0), min(math.ceil(where(slow)), dim - 1)
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        share = min(max((i - low) / (high - low), 0.0), 1.0)
        want = plain * (1 - share) + plain / factor * share
        # powers, one division, two products and a sum in float64: 8 half steps
        assert abs(float(f[i]) - want) <= 8 * 2.0 ** -53 * want, i
        turns = length * plain / (2 * math.pi)
        if turns >= fast:
            assert share == 0.0
        if turns > slow * base ** (2 / dim):  # (more than one whole pair away from the ramp's end)
            assert share < 1.0 and float(f[i]) > plain / factor


@pytest.mark.parametrize("betas", [(1.0, 32.0), (32.0, 0.0), (32.0, -1.0), (math.nan, 1.0), (32.0, math.nan),
                                   (math.inf, 1.0)])
def test_yarn_refuses_ends_out_of_order(betas):
    fast, slow = betas
    with pytest.raises(ValueError, match="beta_fast"):
        prism_amd.rotary_frequencies(64, scaling="yarn", factor=4.0, original_length=8192, beta_fast=fast, beta_slow=slow,
                                     device="cpu")


def fake_calls():
    """(name, call of one fake tensor, its shape): every input that could carry a derivative."""
    bf = torch.bfloat16
    mk = lambda *s, dt=bf: torch.empty(*s, device="cuda", dtype=dt)  # noqa: E731
    x, w = mk(3, 64), mk(64)
    q, freqs, at = mk(1, 2, 9, 64), mk(32, dt=torch.float64), mk(9, dt=torch.int64)
    att = prism_amd.flash_attn_window
    return [("norm x", lambda t: prism_amd.rms_norm(t, w), x), ("norm weight", lambda t: prism_amd.rms_norm(x, t), w),
            ("norm residual", lambda t: prism_amd.rms_norm(x, w, residual=t)[1], x),
            ("norm codes", lambda t: prism_amd.rms_norm_quant(t)[1], x),
            ("rotary q", lambda t: prism_amd.apply_rotary(t, None, freqs, at), q),
            ("rotary k", lambda t: prism_amd.apply_rotary(q, t, freqs, at)[1], q),
            ("rotary freqs", lambda t: prism_amd.apply_rotary(q, None, t, at), freqs),
            ("window q", lambda t: att(t, q, q, 3), q), ("window k", lambda t: att(q, t, q, 3), q),
            ("window v", lambda t: att(q, q, t, 3, return_lse=True)[1], q)]


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(requires_grad):
    import torch.autograd.forward_ad as forward_ad
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        for name, call, t in fake_calls():
            if requires_grad and name in ("norm codes", "rotary freqs"):
                continue  # (refused as such)
            t = t.requires_grad_(requires_grad)
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                        call(dual)
            if not requires_grad:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    torch.func.jvp(call, (t,), (torch.ones_like(t),))
            t.requires_grad_(False)
            assert not call(t).requires_grad  # without a tangent: as ever


def test_vmap_shapes():
    """Every operator under vmap, over any dimension, with inputs that are not
    mapped (fake tensors: shapes and which outputs carry gradients)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    bf = torch.bfloat16
    with FakeTensorMode():
        mk = lambda *s, dt=bf: torch.empty(*s, device="cuda", dtype=dt, requires_grad=dt == bf)  # noqa: E731
        x, w, xs = mk(4, 5, 64), mk(64), mk(5, 4, 64)
        y, h = torch.vmap(lambda a, r, w: prism_amd.rms_norm(a, w, residual=r), in_dims=(0, 1, None))(x, xs, w)
        assert y.shape == h.shape == (4, 5, 64) and y.requires_grad and h.requires_grad
        codes, scales = torch.vmap(prism_amd.rms_norm_quant)(x.detach())
        assert codes.shape == x.shape and codes.dtype == torch.float8_e4m3fn and scales.shape == (4, 5)
        bwd = lambda dy, inv: prism_amd.ops.rms_norm_bwd(dy, None, x.detach()[0], w.detach(), inv, True)  # noqa: E731
        dx, dw = torch.vmap(bwd, in_dims=(1, None))(xs.detach(), mk(5, dt=torch.float32))
        assert dx.shape == x.shape and dw.shape == (4, 64)
        q, k, freqs, at = mk(3, 1, 4, 9, 64), mk(1, 2, 9, 64, 3), mk(32, dt=torch.float64), mk(3, 9, dt=torch.int64)
        a, b = torch.vmap(lambda q, k, at: prism_amd.apply_rotary(q, k, freqs, at), in_dims=(0, 4, 0))(q, k, at)
        assert a.shape == q.shape and b.shape == (3, 1, 2, 9, 64) and b.requires_grad
        at2 = mk(9, 2, dt=torch.int32)
        c = torch.vmap(lambda q: prism_amd.apply_rotary(q, None, freqs, at2, sections=(32, 32)))(q)
        assert c.shape == q.shape
        o, lse = torch.vmap(lambda q, k: prism_amd.flash_attn_window(q, k, k, 5, return_lse=True))(a, b)
        assert o.shape == q.shape and lse.shape == (3, 1, 4, 9) and o.requires_grad and not lse.requires_grad
        with pytest.raises(ValueError, match="vmap"):
            torch.vmap(prism_amd.rms_norm)(x[:0])


@pytest.mark.parametrize("window,sinks,causal,bound", [(5, 0, True, False), (100, 4, True, True), (None, 0, True, True),
                                                       (32, 0, False, False), (33, 0, False, True), (30, 40, True, True),
                                                       (60, 4, True, False), (1 << 62, 1 << 62, False, True)])
@pytest.mark.parametrize("length", [2, 64, 65, 70, 5000])
def test_traced_training_step_keeps_symbolic_lengths(window, sinks, causal, bound, length):
    """One traced program serves every length: a training step's outputs keep the
    symbol as inference's do, and the one choice that depends on the length (what
    the backward keeps) is a bound, not a value."""
    from torch._dynamo.source import ConstantSource
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv
    for grad in (False, True):
        env = ShapeEnv()
        with FakeTensorMode(shape_env=env):
            symbol = env.create_symbol(length, ConstantSource("S"), dynamic_dim=DimDynamic.DYNAMIC)
            S = env.create_symintnode(symbol, hint=length)
            mk = lambda *s, dt=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dt,  # noqa: E731
                                                           requires_grad=grad and dt == torch.bfloat16)  # noqa: B023
            q, x, f, at = mk(2, 4, S, 64), mk(S, 64), mk(32, dt=torch.float64), mk(S, dt=torch.int64)
            o, lse = prism_amd.flash_attn_window(q, q, q, window, sinks=sinks, causal=causal, return_lse=True)
            sizes = [o.shape[2], lse.shape[2], prism_amd.rms_norm(x).shape[0], prism_amd.apply_rotary(q, q, f, at)[1].shape[2]]
        assert all(isinstance(s, torch.SymInt) and s.node.expr == symbol for s in sizes), sizes
        guards = {str(g.expr).replace(str(symbol), "S") for g in env.guards}
        assert guards <= ({"S <= 64" if length <= 64 else "S > 64"} if grad and bound else set()), guards


def test_what_the_backward_keeps_goes_by_one_bound():
    """The rule in use (few keys at any length, or a length of 64 at most) is the
    C function's at every length."""
    lib = prism_amd._lib.load()
    for causal in (0, 1):
        for window in (1, 2, 31, 32, 33, 60, 63, 64, 65, 100, 1 << 29):
            for sinks in (0, 1, 4, 5, 30, 63, 64, 65, 1 << 29):
                any_length = lib.prism_window_rest(1 << 40, window, sinks, causal)
                for Sk in (0, 1, 2, 31, 32, 33, 62, 63, 64, 65, 66, 99, 100, 129, 5000):
                    assert lib.prism_window_rest(Sk, window, sinks, causal) == (any_length and Sk > 64)


def test_adapter_keeps_no_positions():
    """Inference mode, then training on the same grid; and nothing of a call stays."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    freqs, _ = prism_amd.rotary_frequencies(64, sections=(24, 20, 20), device="cpu")
    with FakeTensorMode() as mode:
        m = prism_amd.DynamicBlockSparseAttention(rotary_freqs=mode.from_tensor(freqs).to("cuda"), rotary_sections=(24, 20, 20))
        before = dict(vars(m))
        q = torch.empty(1, 2, 24, 64, device="cuda", dtype=torch.bfloat16)
        with torch.inference_mode():
            m._rotate(q, q, (2, 3, 4))
        a, b = m._rotate(q.clone().requires_grad_(True), q, (2, 3, 4))
        assert a.requires_grad and b.requires_grad
        assert vars(m) == before


def bwd_workspace(B, Hq, Hk, S, D, window, sinks, causal=1, lens=0, Sk=None):
    """Bytes that the window backward's plan asks for, and those of its eight tensors."""
    floats = ctypes.c_int64()
    lib = prism_amd._lib.load()
    assert lib.prism_window_bwd_plan(B, Hq, Hk, S, Sk or S, D, window, sinks, causal, lens, ctypes.byref(floats)) == 0
    return 4 * floats.value, 2 * B * D * 4 * (Hq * S + Hk * (Sk or S))


@pytest.mark.parametrize("case", [(2, 16, 4, 4096, 64, 1024, 4), (16, 32, 8, 2048, 64, 1024, 4), (24, 16, 16, 4096, 64, 1024, 4),
                                  (24, 16, 16, 16384, 64, 4096, 4), (48, 40, 5, 32768, 64, 1024, 4),
                                  (16, 32, 8, 2048, 128, 1024, 4), (3, 9, 9, 5000, 64, 300, 0)])
def test_lengths_take_no_more_workspace(case):
    """What the sequences' lengths are stands on the device: a call that passes them
    is cut as one without, not by a guess of how much of the batch is padding."""
    full, _ = bwd_workspace(*case)
    assert bwd_workspace(*case, lens=1)[0] <= 2 * full


def test_many_sinks_beside_a_narrow_window_take_a_bounded_workspace():
    """Two rounds of pieces for the sinks' lists (67 MB at D = 128, 50 at 64) and the
    cut of the last round, whatever the lengths: within the tensors and 128 MiB,
    and within 256 MiB."""
    for B in (1, 2, 8, 48):
        for Hq, Hk in ((1, 1), (8, 1), (8, 8), (40, 5), (32, 8), (40, 40)):
            for S in (1000, 4096, 16384, 75600, 131072, 300000):
                for D in (64, 128):
                    for window in (1, 64, 256, 1024):
                        for sinks in (128, 640, 1000, 3600, 20000):
                            for causal in (0, 1):
                                work, tensors = bwd_workspace(B, Hq, Hk, S, D, window, sinks, causal)
                                assert work <= min(tensors + (1 << 27), 1 << 28), (B, Hq, Hk, S, D, window, sinks, causal, work)


def test_launches_of_too_many_tiles_are_refused():
    """A launch holds fewer than 2^32 threads (before any launch: status 1, and no
    memory is touched)."""
    lib, one = prism_amd._lib.load(), ctypes.c_void_p(16)
    st = (ctypes.c_int64 * 24)(*[64] * 24)
    shape = lambda B, Sq: (1, B, 1, 1, Sq, 9, 64, st, 3, 0, 1, None, None, 0.1)  # noqa: E731
    for B in (1 << 24, 1 << 30):
        assert lib.prism_window_token(one, one, one, *shape(B, 1), one, None, None, 1, None, None, None) == 1
        assert b"too many" in lib.prism_last_error()
        assert lib.prism_window_fwd(one, one, one, *shape(B, 40), one, None, None, one, None) == 1
        assert b"too many" in lib.prism_last_error()
        assert lib.prism_window_bwd(one, one, one, one, one, None, one, *shape(B, 40), one, one, one, one, one, None) == 1
        assert b"too many" in lib.prism_last_error()
    assert lib.prism_window_token(one, one, one, *shape(1 << 21, 1), one, None, None, 2, one, one, None) == 1
    assert b"too many" in lib.prism_last_error()
