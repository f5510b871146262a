"""The layer's operators as they are used together: residual addition and norm,
projections, rotary positions and attention, forward and backward; a stream's
prompt and its single tokens over a cache; rotary positions inside the
block-sparse adapter."""
import math

import pytest
import torch
import torch.nn.functional as F

import prism_amd
from tests.test_gpu_window import seen_mask

pytestmark = pytest.mark.gpu


def plain_layer(x, r, w, wq, wk, wv, freqs, at, window, sinks, Hq, Hk, D):
    """The layer in the given dtype's plain torch operations (float64)."""
    B, S, _ = x.shape
    h = x + r
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w
    heads = lambda t, H: t.view(B, S, H, D).transpose(1, 2)  # noqa: E731
    q, k, v = heads(y @ wq.t(), Hq), heads(y @ wk.t(), Hk), heads(y @ wv.t(), Hk)

    def turn(t):
        a = at.to(t.dtype)[:, None] * freqs
        t1, t2 = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([t1 * a.cos() - t2 * a.sin(), t1 * a.sin() + t2 * a.cos()], -1)

    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(Hq // Hk, 1) for t in (k, v))
    m = seen_mask(B, S, S, window, sinks, True, None, None)[:, None]
    p = torch.softmax((q @ k.transpose(-1, -2) * D ** -0.5).masked_fill(~m, -math.inf), -1)
    return (p @ v).transpose(1, 2).reshape(B, S, Hq * D), h


def test_layer_forward_and_backward():
    """Norm-wise: five roundings of the type on the way to the output (y, the
    projections, the turned q and k, P, o), each at most u = 2^-8 relative; those
    before the softmax reach o through scores of size ~3, times at most 4: 20 u.
    The backward has as many again on top of the forward's: 60 u."""
    torch.manual_seed(1)
    B, S, C, Hq, Hk, D, window, sinks = 2, 210, 384, 6, 2, 64, 50, 4
    dt = torch.bfloat16
    mk = lambda *s, f=1.0: (torch.randn(*s, device="cuda") * f).to(dt)  # noqa: E731
    x, r, w = mk(B, S, C), mk(B, S, C, f=2), (1 + 0.2 * torch.randn(C, device="cuda")).to(dt)
    wq, wk, wv = mk(Hq * D, C, f=C ** -0.5), mk(Hk * D, C, f=C ** -0.5), mk(Hk * D, C, f=C ** -0.5)
    freqs, _ = prism_amd.rotary_frequencies(D)
    at = torch.arange(S, device="cuda")
    do, dh = mk(B, S, Hq * D), mk(B, S, C)

    leaves = [t.clone().requires_grad_(True) for t in (x, r, w, wq, wk, wv)]
    y, h = prism_amd.rms_norm(leaves[0], leaves[2], residual=leaves[1])
    heads = lambda t, H: t.view(B, S, H, D).transpose(1, 2)  # noqa: E731
    q, k, v = heads(F.linear(y, leaves[3]), Hq), heads(F.linear(y, leaves[4]), Hk), heads(F.linear(y, leaves[5]), Hk)
    q, k = prism_amd.apply_rotary(q, k, freqs, at, interleaved=False)
    o = prism_amd.flash_attn_window(q, k, v, window, sinks=sinks)
    assert o.transpose(1, 2).is_contiguous()
    o = o.transpose(1, 2).reshape(B, S, Hq * D)
    got = [o, h, *torch.autograd.grad((o, h), leaves, (do, dh))]

    leaves64 = [t.double().requires_grad_(True) for t in (x, r, w, wq, wk, wv)]
    o64, h64 = plain_layer(*leaves64, freqs, at, window, sinks, Hq, Hk, D)
    want = [o64, h64, *torch.autograd.grad((o64, h64), leaves64, (do.double(), dh.double()))]
    u = torch.finfo(dt).eps / 2
    for i, (a, b) in enumerate(zip(got, want)):
        err = float((a.double() - b).norm() / b.norm())
        assert err <= (20 if i < 2 else 60) * u, (i, err)


def test_stream_over_a_cache():
    """A prompt, then tokens one by one over a cache with room beyond them (NaN
    there), give what the whole sequence gives at once: within both calls'
    rounding of P and o (2 u sum p |v| + u |o| each)."""
    torch.manual_seed(2)
    B, S, n0, Hq, Hk, D, window, sinks = 2, 150, 100, 8, 2, 128, 40, 3
    dt = torch.bfloat16
    q, k, v = (torch.randn(B, S, H, D, device="cuda").to(dt).transpose(1, 2) for H in (Hq, Hk, Hk))
    freqs, amp = prism_amd.rotary_frequencies(D, scaling="ntk", factor=4.0)
    at = torch.arange(S, device="cuda")
    q, k = prism_amd.apply_rotary(q, k, freqs, at, amplitude=amp)
    whole = prism_amd.flash_attn_window(q, k, v, window, sinks=sinks)
    room = torch.full((B, 256, Hk, D), math.nan, device="cuda", dtype=dt)
    kc, vc = room.clone().transpose(1, 2), room.clone().transpose(1, 2)
    kc[:, :, :n0], vc[:, :, :n0] = k[:, :, :n0], v[:, :, :n0]
    lens = torch.full((B,), n0, dtype=torch.int32, device="cuda")
    outs = [prism_amd.flash_attn_window(q[:, :, :n0], kc, vc, window, sinks=sinks, kv_lens=lens)]
    for t in range(n0, S):
        kc[:, :, t], vc[:, :, t] = k[:, :, t], v[:, :, t]
        lens += 1
        outs.append(prism_amd.flash_attn_window(q[:, :, t:t + 1], kc, vc, window, sinks=sinks, kv_lens=lens))
    got = torch.cat(outs, 2)
    u = torch.finfo(dt).eps / 2
    bound = v.abs().amax(2, keepdim=True).double().repeat_interleave(Hq // Hk, 1)
    assert ((got.double() - whole.double()).abs() <= 4 * u * bound).all()


def test_adapter_turns_q_and_k():
    torch.manual_seed(3)
    grid, D = (5, 10, 12), 64
    S = grid[0] * grid[1] * grid[2]
    q, k, v = (torch.randn(1, 2, S, D, device="cuda").to(torch.bfloat16) for _ in range(3))
    sections = (24, 20, 20)
    freqs, _ = prism_amd.rotary_frequencies(D, sections=sections)
    a = prism_amd.DynamicBlockSparseAttention("ivpq", {"sparsity": 0.5}, rotary_freqs=freqs, rotary_sections=sections)
    b = prism_amd.DynamicBlockSparseAttention("ivpq", {"sparsity": 0.5})
    do = torch.randn_like(q)

    def both(m, turn):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        x, y = leaves[0], leaves[1]
        if turn:
            x, y = prism_amd.apply_rotary(x, y, freqs, prism_amd.grid_positions(grid), sections=sections)
        o = m(x, y, leaves[2], grid)
        return [o, *torch.autograd.grad(o, leaves, do)]

    for s, t in zip(both(a, False), both(b, True)):
        assert torch.equal(s, t)
    assert not torch.equal(both(b, False)[0], both(b, True)[0])
    with pytest.raises(ValueError, match="rotary_sections"):
        prism_amd.DynamicBlockSparseAttention(rotary_freqs=freqs)


def test_layer_captured():
    """A stream's step (norm to 8 bits aside, rotary, attention over the cache) in
    one graph, replayed as the stream grows."""
    torch.manual_seed(4)
    B, Hq, Hk, D = 3, 8, 2, 64
    dt = torch.float16
    x, r = torch.randn(B, 1, Hq * D, device="cuda").to(dt), torch.randn(B, 1, Hq * D, device="cuda").to(dt)
    w = torch.ones(Hq * D, device="cuda", dtype=dt)
    kc, vc = (torch.randn(B, Hk, 300, D, device="cuda").to(dt) for _ in range(2))
    freqs, _ = prism_amd.rotary_frequencies(D)
    at = torch.tensor([[100], [200], [5]], device="cuda")
    lens = (at.view(-1) + 1).int()

    def step():
        y, h = prism_amd.rms_norm(x, w, residual=r)
        codes, scales, _ = prism_amd.rms_norm_quant(x, w, residual=r)
        q = prism_amd.apply_rotary(y.view(B, 1, Hq, D).transpose(1, 2), None, freqs, at, interleaved=False)
        return prism_amd.flash_attn_window(q, kc, vc, 64, sinks=4, kv_lens=lens), h, codes.float(), scales

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        x.normal_()
        at += 1
        lens += 1
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
