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
        err = float(((a.double() - b).norm() / b.norm()).detach())
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


def small_layer(x, w, freqs, at, kv):
    y = prism_amd.rms_norm(x, w)
    q = y.view(2, 70, 4, 64).transpose(1, 2)
    q, k = prism_amd.apply_rotary(q, q[:, ::2], freqs, at)
    return prism_amd.flash_attn_window(q, k, kv, 20, sinks=2)


def small_inputs(seed=0):
    torch.manual_seed(seed)
    x, w = torch.randn(2, 70, 256, device="cuda").to(torch.bfloat16), torch.ones(256, device="cuda", dtype=torch.bfloat16)
    kv = torch.randn(2, 2, 70, 64, device="cuda").to(torch.bfloat16)
    return x, w, prism_amd.rotary_frequencies(64)[0], torch.arange(70, device="cuda"), kv


def test_compiled_gives_the_same_bits():
    """Traced whole (no graph break), forward and backward through the operators'
    fake implementations, and run: the eager results."""
    x, w, freqs, at, kv = small_inputs()
    compiled = torch.compile(small_layer, backend="aot_eager", fullgraph=True)
    for grad in (False, True):
        leaves = [t.clone().requires_grad_(grad) for t in (x, w, kv)]
        outs = []
        for f in (small_layer, compiled):
            o = f(leaves[0], leaves[1], freqs, at, leaves[2])
            outs.append([o.detach(), *(torch.autograd.grad(o, leaves, torch.ones_like(o)) if grad else ())])
        assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_output_layouts():
    """The fake implementations promise the layouts that the kernels' outputs have."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    dt = torch.bfloat16
    base = torch.randn(2, 30, 4, 64, device="cuda").to(dt)
    wide = torch.randn(2, 4, 30, 72, device="cuda").to(dt)
    freqs, at = prism_amd.rotary_frequencies(64)[0], torch.arange(30, device="cuda")
    for t in (base.transpose(1, 2), wide[..., :64], wide[..., 3:67], base.permute(0, 3, 1, 2).transpose(2, 3).permute(0, 2, 3, 1),
              torch.randn(2, 4, 30, 128, device="cuda").to(dt)[..., ::2], wide[:, :1, :, 8:].expand(2, 4, 30, 64),
              torch.randn(30, 64, 4, 2, device="cuda").to(dt).permute(3, 2, 0, 1)):
        assert t.shape == (2, 4, 30, 64)
        got = [*prism_amd.apply_rotary(t, t[:, :2], freqs, at), prism_amd.flash_attn_window(t, t, t, 9)]
        with FakeTensorMode() as mode:
            f, ff, fa = (mode.from_tensor(x) for x in (t, freqs, at))
            fake = [*prism_amd.apply_rotary(f, f[:, :2], ff, fa), prism_amd.flash_attn_window(f, f, f, 9)]
        assert [x.stride() for x in got] == [x.stride() for x in fake]
    far = torch.randn(2, 4096, 64, 64, device="cuda").to(dt).permute(1, 2, 0, 3)  # rows 2^24 elements apart
    assert torch.equal(prism_amd.flash_attn_window(far, far, far, 2), prism_amd.flash_attn_window(*[far.contiguous()] * 3, 2))


def test_capture_of_leaves_that_an_eager_graph_holds_is_refused():
    x, w, freqs, at, kv = small_inputs()
    cases = [(w, lambda t: prism_amd.rms_norm(x, t)), (x, lambda t: prism_amd.rms_norm(x, w, residual=t)[0]),
             (kv, lambda t: prism_amd.flash_attn_window(kv, kv, t, 9)), (kv, lambda t: prism_amd.apply_rotary(kv, t, freqs, at)[1])]
    for value, op in cases:
        leaf = value.clone().requires_grad_(True)
        held = op(leaf)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mark = torch.zeros(1, device="cuda")
            with pytest.raises(RuntimeError, match="eager calls"):
                op(leaf)
        assert held.requires_grad and mark.numel() == 1
        ones = torch.ones_like(held.detach())
        del held  # with the eager graph gone the same call is captured, backward and all
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            (got,) = torch.autograd.grad(op(leaf), leaf, ones)
        graph.replay()
        torch.cuda.synchronize()
        (want,) = torch.autograd.grad(op(leaf), leaf, ones)
        assert torch.equal(got, want)


def test_threads_and_streams():
    """Four threads, each with its own stream, inputs and backward pass."""
    import threading
    inputs = [small_inputs(i) for i in range(4)]

    def run(i, out):
        x, w, freqs, at, kv = inputs[i]
        leaves = [t.clone().requires_grad_(True) for t in (x, w, kv)]
        o = small_layer(leaves[0], leaves[1], freqs, at, leaves[2])
        out[i] = [o.detach(), *torch.autograd.grad(o, leaves, torch.ones_like(o))]

    want, got, errors = {}, {}, []
    for i in range(4):
        run(i, want)
    torch.cuda.synchronize()

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    run(i, got)
            s.synchronize()
        except BaseException as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(4):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))


def test_offsets_past_32_bits():
    """Rows, tokens and cache entries whose offsets pass 2^32 bytes and 2^31
    elements: the last ones give what they give alone."""
    dt = torch.bfloat16
    M, N, tail = 1_500_000, 1536, 37
    x = torch.zeros(M, N, device="cuda", dtype=dt)
    x[-tail:] = torch.randn(tail, N, device="cuda")
    w = torch.randn(N, device="cuda").to(dt)
    y, h = prism_amd.rms_norm(x, w, residual=x)
    y2, h2 = prism_amd.rms_norm(x[-tail:], w, residual=x[-tail:])
    assert torch.equal(y[-tail:], y2) and torch.equal(h[-tail:], h2)
    codes, scales = prism_amd.rms_norm_quant(x, w)
    c2, s2 = prism_amd.rms_norm_quant(x[-tail:], w)
    assert torch.equal(codes[-tail:].float(), c2.float()) and torch.equal(scales[-tail:], s2)
    leaves, few = [t.clone().requires_grad_(True) for t in (x, w)], [t.clone().requires_grad_(True) for t in (x[-tail:], w)]
    dx, dw = torch.autograd.grad(prism_amd.rms_norm(leaves[0], leaves[1]), leaves, x)
    dx2, dw2 = torch.autograd.grad(prism_amd.rms_norm(few[0], few[1]), few, x[-tail:])
    assert torch.equal(dx[-tail:], dx2)
    # the zero rows add nothing; fp32 sums in another order, rounded once more each
    assert ((dw.float() - dw2.float()).abs() <= 2 * torch.finfo(dt).eps * dw2.float().abs() + 2.0 ** -16).all()
    del x, y, h, codes, leaves, dx
    S, H, D = 2_400_000, 8, 128
    cache = torch.zeros(2, 1, S, H, D, device="cuda", dtype=dt)
    cache[:, :, :3] = torch.randn(2, 1, 3, H, D, device="cuda")
    cache[:, :, -6000:] = torch.randn(2, 1, 6000, H, D, device="cuda")
    k, v = cache[0].transpose(1, 2), cache[1].transpose(1, 2)
    window, sinks = 5000, 3
    near = torch.cat([cache[:, :, :3], cache[:, :, -6000:]], 2)  # the same keys without the middle
    k2, v2 = near[0].transpose(1, 2), near[1].transpose(1, 2)
    for n in (1, 300):
        q = torch.randn(1, H, n, D, device="cuda").to(dt)
        o = prism_amd.flash_attn_window(q, k, v, window, sinks=sinks)
        o2 = prism_amd.flash_attn_window(q, k2, v2, window, sinks=sinks)
        # other tile borders: two roundings of P and o each
        assert ((o.float() - o2.float()).abs() <= 2 * torch.finfo(dt).eps * v2.abs().max().float()).all()
    leaves, few = [t.detach().requires_grad_(True) for t in (q, k, v)], [t.detach().requires_grad_(True) for t in (q, k2, v2)]
    got = torch.autograd.grad(prism_amd.flash_attn_window(*leaves, window, sinks=sinks), leaves, q)
    want = torch.autograd.grad(prism_amd.flash_attn_window(*few, window, sinks=sinks), few, q)
    at = torch.cat([torch.arange(3, device="cuda"), torch.arange(S - 6000, S, device="cuda")])
    for i in (1, 2):
        a, b = got[i][:, :, at].float(), want[i].float()
        assert (a - b).norm() <= 8 * torch.finfo(dt).eps * b.norm()
        assert (got[i][:, :, 3:S - 6000] == 0).all()
    assert (got[0].float() - want[0].float()).norm() <= 8 * torch.finfo(dt).eps * want[0].float().norm()
    # rotary: the last token of a long, wide sequence
    freqs = prism_amd.rotary_frequencies(D)[0]
    pos = torch.arange(S, device="cuda")
    r = prism_amd.apply_rotary(k, None, freqs, pos)
    assert torch.equal(r[:, :, -50:], prism_amd.apply_rotary(k[:, :, -50:], None, freqs, pos[-50:]))
