"""Corners of the layer's operators on the GPU: transforms, streams, ranges of
float16, sizes of launches and workspaces."""
import pytest
import torch

import prism_amd

pytestmark = pytest.mark.gpu


def randn(*shape, dt=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dt)


def test_vmap_gives_the_bits_of_a_loop():
    """Forward and backward over a mapped dimension, with inputs and leaves that
    are not mapped, and backward passes mapped over the outputs' gradients."""
    x, r, w = randn(4, 5, 64, seed=1), randn(5, 4, 64, seed=2), randn(64, seed=3)
    q, kv, at = randn(4, 1, 4, 9, 64, seed=4), randn(1, 2, 9, 64, 4, seed=5), torch.arange(36, device="cuda").view(4, 9)
    freqs = prism_amd.rotary_frequencies(64)[0]

    def layer(x, r, w, q, kv, at):
        y, h = prism_amd.rms_norm(x, w, residual=r)
        q, k = prism_amd.apply_rotary(q, kv, freqs, at)
        return y, h, prism_amd.flash_attn_window(q, k, kv, 5, sinks=1)

    dims = (0, 1, None, 0, 4, 0)
    runs = []
    for mapped in (True, False):
        leaves = [t.clone().requires_grad_(True) for t in (x, r, w, q, kv)]
        if mapped:
            out = torch.vmap(layer, in_dims=dims)(*leaves, at)
        else:
            each = [layer(*[t if d is None else t.select(d, i) for t, d in zip((*leaves, at), dims)]) for i in range(4)]
            out = [torch.stack(ts) for ts in zip(*each)]
        runs.append([*out, *torch.autograd.grad(out, leaves, [randn(*o.shape, seed=9) for o in out])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))

    for out_dtype in (torch.float8_e4m3fn, torch.int8):
        got = torch.vmap(lambda t: prism_amd.rms_norm_quant(t, w, out_dtype=out_dtype))(x)  # noqa: B023
        each = [prism_amd.rms_norm_quant(t, w, out_dtype=out_dtype) for t in x]
        assert all(torch.equal(a.float(), torch.stack([e[i].float() for e in each])) for i, a in enumerate(got))
    leaves = [t.clone().requires_grad_(True) for t in (x[0], w, q[0])]
    y = prism_amd.rms_norm(leaves[0], leaves[1])
    o = prism_amd.flash_attn_window(*[prism_amd.apply_rotary(leaves[2], None, freqs, at[0])] * 3, 5)
    for out, ins in ((y, leaves[:2]), (o, leaves[2:])):
        d = randn(3, *out.shape, seed=7)
        got = torch.vmap(lambda d: torch.autograd.grad(out, ins, d, retain_graph=True))(d)  # noqa: B023
        each = [torch.autograd.grad(out, ins, d[i], retain_graph=True) for i in range(3)]
        assert all(torch.equal(a, torch.stack(b)) for a, b in zip(got, zip(*each)))


def test_tangents_are_refused():
    import torch.autograd.forward_ad as forward_ad
    x = randn(3, 64)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: prism_amd.rms_norm(t), (x,), (torch.ones_like(x),))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        prism_amd.rms_norm(forward_ad.make_dual(x, x))
    with pytest.raises(RuntimeError, match="functorch"):  # (torch's own refusal of C++ nodes)
        torch.func.grad(lambda t: prism_amd.rms_norm(t).float().sum())(x)


def test_compiled_training_step_serves_every_length():
    """Compiled once with dynamic lengths: one program, the eager bits, forward and
    backward, at lengths on one side of the bound that decides what is kept."""
    torch._dynamo.reset()
    freqs = prism_amd.rotary_frequencies(64)[0]

    def step(q, kv, w, at):
        q, k = prism_amd.apply_rotary(q, kv, freqs, at)
        return prism_amd.rms_norm(prism_amd.flash_attn_window(q, k, kv, 100, sinks=4), w)

    fast = torch.compile(step, backend="aot_eager", dynamic=True, fullgraph=True)
    for n in (70, 71, 333, 128):
        args = [randn(1, 4, n, 64, seed=n), randn(1, 2, n, 64, seed=n + 1), randn(64, seed=2)]
        runs = []
        for f in (step, fast):
            leaves = [t.clone().requires_grad_(True) for t in args]
            with torch.compiler.set_stance("default" if n == 70 else "fail_on_recompile"):
                o = f(*leaves, torch.arange(n, device="cuda"))
            runs.append([o.detach(), *torch.autograd.grad(o, leaves, randn(*o.shape, seed=5))])
        assert all(torch.equal(a, b) for a, b in zip(*runs)), n


def test_adapter_positions_on_two_streams():
    """A call behind a long queue of work on one stream does not hold up, or feed,
    one of the same grid on another."""
    sections = (24, 20, 20)
    freqs, _ = prism_amd.rotary_frequencies(64, sections=sections)
    m = prism_amd.DynamicBlockSparseAttention(rotary_freqs=freqs, rotary_sections=sections)
    grids = [(3, 10, 12), (5, 6, 12)]
    q, k = randn(1, 2, 360, 64, seed=1), randn(1, 2, 360, 64, seed=2)
    want = [prism_amd.apply_rotary(q, k, freqs, prism_amd.grid_positions(g), sections=sections) for g in grids]
    busy, work = torch.cuda.Stream(), randn(4096, 4096)
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(busy):
            for _ in range(20):
                work = (work @ work).clamp(-1, 1)
            first = m._rotate(q, k, grids[i % 2])
        got.append((i % 2, m._rotate(q, k, grids[i % 2])))
        got.append((i % 2, first))
    torch.cuda.synchronize()
    for g, (a, b) in got:
        assert torch.equal(a, want[g][0]) and torch.equal(b, want[g][1])


def test_adapter_positions_in_a_graph():
    """The first call on a grid is captured, the next ones run eagerly before the
    graph's first replay."""
    sections = (24, 20, 20)
    freqs, _ = prism_amd.rotary_frequencies(64, sections=sections)
    m = prism_amd.DynamicBlockSparseAttention(rotary_freqs=freqs, rotary_sections=sections)
    q, k = randn(1, 2, 360, 64, seed=1), randn(1, 2, 360, 64, seed=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m._rotate(q, k, (3, 10, 12))
    want = prism_amd.apply_rotary(q, k, freqs, prism_amd.grid_positions((3, 10, 12)), sections=sections)
    assert all(torch.equal(a, b) for a, b in zip(m._rotate(q, k, (3, 10, 12)), want))
    for i in range(3):
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(m._rotate(q, k, (3, 10, 12)), got))


# ------------------------------------------------------------------ float16's range
def sink_and_tail(Sq, Sk, D, gap, dt, Hq=1):
    """One key whose score is `gap` (about) above all the others', which are equal;
    its value is 0, theirs 1 (and 0.5 in every other channel)."""
    q, k = torch.zeros(1, Hq, Sq, D, device="cuda", dtype=dt), torch.zeros(1, 1, Sk, D, device="cuda", dtype=dt)
    v = torch.ones(1, 1, Sk, D, device="cuda", dtype=dt)
    v[..., ::2] = 0.5
    q[..., 0], k[0, 0, 0, 0], v[0, 0, 0] = 4.0, gap / 4, 0
    return q, k, v


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Sq,Sk,D,gap,Hq", [(1, 131073, 64, 17.2, 1), (1, 131073, 128, 17.2, 32), (1, 65001, 64, 17.0, 4),
                                            (200, 65001, 64, 17.0, 4), (300, 30001, 128, 16.0, 2), (1, 400, 64, 11.0, 1),
                                            (130, 400, 64, 11.0, 1), (1, 1000, 128, 17.5, 2), (200, 1000, 64, 17.5, 2)])
def test_long_tails_below_one_large_score(Sq, Sk, D, gap, Hq, dt):
    """A weight far below the largest still counts with its own precision: each P off
    by u of itself (no steps of float16's subnormals: 2^-26 of the largest is 18.0
    nats), all in one direction here; fp32 scores and exponentials (E = (D + 2) 2^-24
    of a score of `gap`, and 2^-22), sums of n terms, o's rounding u (its values
    are at most 1)."""
    q, k, v = sink_and_tail(Sq, Sk, D, gap, dt, Hq)
    o, lse = prism_amd.flash_attn_window(q, k, v, None, causal=False, sm_scale=1.0, return_lse=True)
    score = float(q[0, 0, 0, 0]) * float(k[0, 0, 0, 0])
    tail = torch.tensor(-score, dtype=torch.float64).exp() * (Sk - 1)
    want = (tail / (1 + tail)) * v[:, :, -1:].double()
    u = torch.finfo(dt).eps / 2
    rel = u * 1.01 + 2 * ((D + 2) * 2.0 ** -24 * score + 2.0 ** -22) + Sk * 2.0 ** -24
    tol = (rel + u) * want + torch.finfo(dt).smallest_normal * u
    assert ((o.double() - want).abs() <= tol).all(), (float(o.double().amax()), float(want.amax()))
    assert (lse.double() - (score + float(torch.log1p(tail)))).abs().max() <= 2 * (D + 2) * 2.0 ** -24 * score + 2.0 ** -20


def test_scores_that_rise_by_less_than_the_margin():
    """Each tile's largest score a little above the last one's: float16's P goes to
    2^15 and no further, with values up to the type's largest."""
    D, Sk = 64, 64 * 40
    for step in (0.5, 1.5, 2.07, 2.09, 4.0):  # nats per tile, around the margin of 3 bits
        q, k = torch.zeros(1, 1, 130, D, device="cuda").half(), torch.zeros(1, 1, Sk, D, device="cuda").half()
        q[..., 0] = 1
        k[0, 0, :, 0] = (torch.arange(Sk, device="cuda") // 64) * step
        v = torch.full((1, 1, Sk, D), 60000.0, device="cuda").half()
        for n in (1, 130):
            o = prism_amd.flash_attn_window(q[:, :, :n], k, v, None, causal=False, sm_scale=1.0)
            assert ((o.float() / v[0, 0, 0, 0].float() - 1).abs() <= 2.0 ** -9).all(), step


def gradients64(q, k, v, do, mask):
    """(dq, dk, dv) of softmax attention over a [Sq, Sk] mask, float64, one key head per query head."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    scale = q.shape[-1] ** -0.5
    P = torch.softmax((q @ k.transpose(-1, -2).contiguous() * scale).masked_fill(~mask, -torch.inf), -1)
    dP = do @ v.transpose(-1, -2).contiguous()
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    return scale * (dS @ k), scale * (dS.transpose(-1, -2).contiguous() @ q), P.transpose(-1, -2).contiguous() @ do


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("Sq,Sk,window", [(700, 5000, None), (5000, 5000, 4096), (40, 8000, None)])
def test_float16_gradients_of_small_outputs(Sq, Sk, window, size, D):
    """Norm-wise, what float16's range costs is what the results' own rounding
    costs: independent roundings (P, dS, lse, the rest of o) of at most u each, in
    quadrature 2 u, and the results' rounding with its subnormal steps (rounding the
    exact results), a tenth more for the steps of dS far below them."""
    q, k, v, do = (randn(1, 2, n, D, dt=torch.float16, seed=i) for i, n in enumerate((Sq, Sk, Sk, Sq)))
    do = (do.float() * size).half()
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(prism_amd.flash_attn_window(*leaves, window), leaves, do)
    p = torch.arange(Sq, device="cuda")[:, None] + Sk - Sq
    j = torch.arange(Sk, device="cuda")[None]
    want = gradients64(*[t.detach() for t in leaves], do, (j <= p) & (j > p - (window or 1 << 30)))
    u = torch.finfo(torch.float16).eps / 2
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        err, own = float((a.double() - b).norm()), float((b.half().double() - b).norm())
        assert err <= 2 * u * float(b.norm()) + 1.1 * own, name


def test_float16_gradients_of_large_outputs():
    """dS of several hundred is still finite and right."""
    q, k, v = (randn(1, 2, 300, 64, dt=torch.float16, seed=i) for i in range(3))
    do = (randn(1, 2, 300, 64, dt=torch.float16, seed=4).float() * 64).half()
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(prism_amd.flash_attn_window(*leaves, None, causal=False), leaves, do)
    want = gradients64(*[t.detach() for t in leaves], do, torch.ones(300, 300, device="cuda", dtype=torch.bool))
    for a, b in zip(got, want):  # (four roundings in quadrature and the results' own)
        assert (a.double() - b).norm() <= 3 * torch.finfo(torch.float16).eps / 2 * b.norm()


@pytest.mark.parametrize("case", [(1, 2, 1, 3000, 128, 50, 700, True), (1, 4, 4, 2500, 64, 40, 1500, True),
                                  (2, 20, 20, 1500, 128, 30, 900, True), (1, 3, 3, 2000, 128, 64, 640, False),
                                  (1, 60, 60, 700, 64, 20, 500, True), (1, 300, 300, 400, 128, 20, 200, True)],
                         ids=lambda c: "-".join(str(x) for x in c))
def test_gradients_of_many_sinks_beside_a_narrow_window(case):
    """The sinks' lists in many pieces, in few, and whole."""
    from tests.test_gpu_window_bwd import check
    B, Hq, Hk, S, D, window, sinks, causal = case
    q, k, v, do = (randn(B, H, S, D, seed=i) for i, H in enumerate((Hq, Hk, Hk, Hq)))
    check(q, k, v, do, window, sinks=sinks, causal=causal)


# ------------------------------------------------------------------ sizes of launches
@pytest.mark.parametrize("dt,code,M,N,groups", [
    (torch.bfloat16, 1, 1024, 1536, 256), (torch.bfloat16, 1, 1024, 1535, 512), (torch.float32, 0, 90, 1024, 23),
    (torch.float32, 0, 90, 1028, 90), (torch.float16, 2, 7, 2048, 2), (torch.float16, 2, 7, 2056, 7), (torch.bfloat16, 1, 1, 300, 1),
    (torch.bfloat16, 1, 3000, 2048, 512), (torch.bfloat16, 1, 9, 256, 3), (torch.bfloat16, 1, 300, 9000, 256)])
def test_norm_backward_starts_no_workgroup_without_a_row(dt, code, M, N, groups):
    """A workgroup of the backward leaves its sums in a row of the workspace: the
    rows past those that have rows of the input to add stay as they were."""
    import ctypes
    lib = prism_amd._lib.load()
    parts = ctypes.c_int()
    assert lib.prism_rms_norm_parts(M, N, ctypes.byref(parts)) == 0 and parts.value >= groups
    x, dy, w = randn(M, N, dt=dt, seed=1), randn(M, N, dt=dt, seed=2), randn(N, dt=dt, seed=3)
    inv = torch.rsqrt((x.float() ** 2).mean(-1) + 1e-6)
    partial = torch.full((parts.value, N), 7.0, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    rc = lib.prism_rms_norm_bwd(dy.data_ptr(), N, None, 0, x.data_ptr(), N, w.data_ptr(), code, code, M, N, inv.data_ptr(),
                                dx.data_ptr(), partial.data_ptr(), parts.value, dw.data_ptr(),
                                torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert (partial[groups:] == 7.0).all() and not (partial[:groups] == 7.0).all(1).any()
    # each product and sum in fp32: (M + 4) 2^-24 of the terms' magnitudes, and dw's own rounding
    want = (dy.double() * x.double() * inv.double()[:, None]).sum(0)
    size = (dy.double() * x.double() * inv.double()[:, None]).abs().sum(0)
    assert ((dw.double() - want).abs() <= (M + 4) * 2.0 ** -24 * size + torch.finfo(dt).eps / 2 * want.abs() + 2.0 ** -25).all()


def test_more_rows_than_a_launch_holds():
    """2^22 rows of a thousand threads each and more, 2^24 workgroups of tokens and
    more: rows at the borders and the end give what they give alone."""
    dt, M, N = torch.bfloat16, (1 << 22) + 5, 1025
    x, r, w = torch.zeros(M, N, device="cuda", dtype=dt), torch.zeros(M, N, device="cuda", dtype=dt), randn(N, seed=1)
    some = [slice(0, 3), slice((1 << 21) - 2, (1 << 21) + 3), slice((1 << 22) - 2, M)]
    for i, s in enumerate(some):
        x[s], r[s] = randn(s.stop - s.start, N, seed=i), randn(s.stop - s.start, N, seed=i + 9)
    y, h, _, inv = prism_amd.ops.rms_norm(x, r, w, 1e-6, want_inv=True)
    for s in some:
        y2, h2, _, inv2 = prism_amd.ops.rms_norm(x[s], r[s], w, 1e-6, want_inv=True)
        assert torch.equal(y[s], y2) and torch.equal(h[s], h2) and torch.equal(inv[s], inv2)
    del y, h
    codes, scales = prism_amd.rms_norm_quant(x, w, out_dtype=torch.int8)
    for s in some:
        c2, s2 = prism_amd.rms_norm_quant(x[s], w, out_dtype=torch.int8)
        assert torch.equal(codes[s], c2) and torch.equal(scales[s], s2)
    del x, r, codes
    S, D = (1 << 25) + 3, 129  # (two tokens a workgroup)
    q, at, freqs = torch.zeros(1, 1, S, D, device="cuda", dtype=dt), torch.arange(S, device="cuda"), prism_amd.rotary_frequencies(2)[0]
    some = [slice(0, 3), slice((1 << 24) - 3, (1 << 24) + 3), slice(S - 5, S)]
    for i, s in enumerate(some):
        q[:, :, s] = randn(1, 1, s.stop - s.start, D, seed=i)
    o = prism_amd.apply_rotary(q, None, freqs, at)
    for s in some:
        assert torch.equal(o[:, :, s], prism_amd.apply_rotary(q[:, :, s], None, freqs, at[s]))


def test_kernel_timing_sees_backward_launches():
    """Forward and backward launches, by entry point, on the stream they run on;
    nothing is left of the block outside it."""
    from prism_amd import ops
    freqs, at = prism_amd.rotary_frequencies(64)[0], torch.arange(70, device="cuda")
    x, w, kv = randn(2, 70, 256, seed=1), randn(256, seed=2), randn(2, 2, 70, 64, seed=3)

    def forward(grad):
        leaves = [t.clone().requires_grad_(grad) for t in (x, w, kv)]
        q = prism_amd.rms_norm(leaves[0], leaves[1]).view(2, 70, 4, 64).transpose(1, 2)
        q, k = prism_amd.apply_rotary(q, leaves[2], freqs, at)
        return leaves, prism_amd.flash_attn_window(q, k, k, 20, sinks=2)

    def step():
        leaves, o = forward(True)
        return [o.detach(), *torch.autograd.grad(o, leaves, torch.ones_like(o))]

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with ops.kernel_timing() as tm, torch.cuda.stream(stream):
        got = [step() for _ in range(3)]
        forward(False)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    calls = {name: n for name, (n, ms) in ops.summarize(tm).items() if ms > 0}
    assert calls == {"prism_rms_norm": 4, "prism_rms_norm_bwd": 3, "prism_rotary": 7, "prism_window_fwd": 4, "prism_window_bwd": 3}
    with ops.kernel_timing() as tm:
        leaves, o = forward(True)
    grads = torch.autograd.grad(o, leaves, torch.ones_like(o))
    assert all(torch.equal(a, b) for a, b in zip(grads, want[1:]))
    torch.cuda.synchronize()
    assert {name: n for name, (n, _) in ops.summarize(tm).items()} == {"prism_rms_norm": 1, "prism_rotary": 1, "prism_window_fwd": 1}
