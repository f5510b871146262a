"""The operators of packed batches and paged caches together, as a program uses them:
a layer's training step over packed documents, prompts and decoding steps of a server;
and their corners: transforms, compiled programs, streams, graphs, sizes of tensors and
launches."""
import math

import pytest
import torch

import prism_amd
from tests.test_gpu_packed import cu
from tests.test_gpu_paged import ints, of_cache, table_for

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, dt=torch.bfloat16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dt)


def heads(t):  # [T, H, D] as [1, H, T, D] and back: views
    return t.transpose(0, 1)[None]


def tokens(t):
    return t[0].transpose(0, 1)


def places(lens):
    return torch.cat([torch.arange(n, device=DEV) for n in lens])


def layer(q, k, v, wq, wk, freqs, at, bounds):
    q, k = prism_amd.qk_norm_rotary(heads(q), heads(k), wq, wk, freqs, at, interleaved=False)
    return prism_amd.flash_attn_packed(tokens(q), tokens(k), v, bounds)


def layer64(q, k, v, wq, wk, freqs, at, lens):
    """The same in float64, sequence by sequence, with its gradients' graph."""
    def turn(x, w):
        x = x * (x.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        a, b = x.chunk(2, -1)
        c, s = ((at.double()[:, None] * freqs)[:, None].cos(), (at.double()[:, None] * freqs)[:, None].sin())
        return torch.cat([a * c - b * s, a * s + b * c], -1)
    q, k, G, out = turn(q, wq), turn(k, wk), q.shape[1] // k.shape[1], []
    for x, y, z in zip(q.split(lens), k.split(lens), v.split(lens)):
        n = len(x)
        y, z = (t.repeat_interleave(G, 1).transpose(0, 1) for t in (y, z))
        s = (x.transpose(0, 1) @ y.transpose(1, 2).contiguous() / math.sqrt(q.shape[-1])).masked_fill(
            ~torch.ones(n, n, dtype=torch.bool, device=DEV).tril(), -math.inf)
        out.append((torch.softmax(s, -1) @ z).transpose(0, 1))
    return torch.cat(out)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_training_step_over_packed_documents(dt):
    """Values and all gradients of norm, positions and attention in a row.  Norm-wise,
    with u half a step of the type: q and k, rounded once, move each score (fan of some
    units) by u and so P by a few u; P, dS, o and dy rounded: 8 u."""
    lens, Hq, Hk, D = [130, 1, 77, 300], 8, 2, 128
    T, u = sum(lens), torch.finfo(dt).eps / 2
    args = [randn(T, Hq, D, dt=dt, seed=1), randn(T, Hk, D, dt=dt, seed=2), randn(T, Hk, D, dt=dt, seed=3),
            (torch.rand(D, device=DEV) + 0.5).to(dt), (torch.rand(D, device=DEV) + 0.5).to(dt)]
    freqs, _ = prism_amd.rotary_frequencies(D)
    at, do = places(lens), randn(T, Hq, D, dt=dt, seed=4)
    leaves = [t.clone().requires_grad_(True) for t in args]
    o = layer(*leaves, freqs, at, cu(lens))
    got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
    exact = [t.double().requires_grad_(True) for t in args]
    want = layer64(*exact, freqs, at, lens)
    want = [want.detach(), *torch.autograd.grad(want, exact, do.double())]
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 8 * u * b.norm()
    assert got[0].is_contiguous()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_server(bits):
    """Prompts packed and appended; a second part of them over its cached first part;
    decoding steps: every output against float64 attention over what the cache holds."""
    Hq, Hk, D, page, dt = 8, 2, 128, 16, torch.bfloat16
    freqs, _ = prism_amd.rotary_frequencies(D)
    parts, steps = [[40, 7, 90], [25, 60, 1]], 3
    final = [sum(p[b] for p in parts) + steps for b in range(3)]
    table, pages = table_for(final, page)
    kc, vc = prism_amd.paged_cache(pages, page, Hk, D, bits=bits)

    def attend64(q, lens, new):
        K, V = of_cache(kc, D), of_cache(vc, D)
        out = []
        for b, (L, n) in enumerate(zip(lens, new)):
            at = torch.arange(L, device=DEV)
            k, v = (c[table[b, at // page].long(), :, at % page].permute(1, 0, 2).repeat_interleave(Hq // Hk, 0) for c in (K, V))
            s = q[sum(new[:b]):sum(new[:b]) + n].double().transpose(0, 1) @ k.transpose(1, 2).contiguous() / math.sqrt(D)
            s = s.masked_fill(at > torch.arange(L - n, L, device=DEV)[:, None], -math.inf)
            out.append((torch.softmax(s, -1) @ v).transpose(0, 1))
        return torch.cat(out)

    lens = [0, 0, 0]
    for step, new in enumerate(parts + [[1, 1, 1]] * steps):
        T = sum(new)
        lens = [a + n for a, n in zip(lens, new)]
        at = torch.cat([torch.arange(L - n, L, device=DEV) for L, n in zip(lens, new)])
        q, k, v = (randn(T, H, D, seed=10 * step + H + i) for i, H in enumerate((Hq, Hk, Hk)))
        q = tokens(prism_amd.apply_rotary(heads(q), None, freqs, at))
        before = [of_cache(c, D) for c in (kc, vc)]
        if len(new) * 1 == T:
            prism_amd.append_paged(k, v, kc, vc, table, ints(lens), freqs=freqs)
            o = prism_amd.flash_attn_paged(q, kc, vc, table, ints(lens))
        else:
            prism_amd.append_paged(k, v, kc, vc, table, ints(lens), cu_seqlens=cu(new), freqs=freqs)
            kk, vv = prism_amd.gather_paged(kc, vc, table, cu(lens), sum(lens), head_dim=D)
            o = prism_amd.flash_attn_packed(q, kk, vv, cu(new), cu_seqlens_k=cu(lens))
        want = attend64(q, lens, new)
        assert (o.double() - want).norm() <= 3 * 2.0 ** -8 * want.norm()
        changed = sum((a != of_cache(c, D)).any(-1).sum().item() for a, c in zip(before, (kc, vc)))
        assert changed <= 2 * Hk * T  # (the new places, and no others)
    if bits == 16:  # the appended keys are those that the rotation gives, but for roundings
        k = tokens(prism_amd.apply_rotary(heads(k), heads(k), freqs, at)[1])
        for b, L in enumerate(lens):
            held = kc[int(table[b, (L - 1) // page]), :, (L - 1) % page]
            assert (held.float() - k[b].float()).abs().max() <= 2.0 ** -7 * k[b].float().abs().max()


def test_decoding_steps_in_a_graph():
    """One captured step, replayed with eager work and synchronizations in between: the
    caches and outputs of eager steps, bit for bit; both widths, lengths that grow."""
    Hq, Hk, D, page, B = 8, 2, 128, 16, 3
    freqs, _ = prism_amd.rotary_frequencies(D)
    for bits in (16, 4):
        table, pages = table_for([900, 60, 40], page)
        lens = ints([800, 30, 15])
        q, k, v = (randn(B, H, D, seed=H + i) for i, H in enumerate((Hq, Hk, Hk)))
        w = torch.ones(D, device=DEV)
        own = prism_amd.paged_cache(pages, page, Hk, D, bits=bits)
        for c in own:
            c.random_(0, 100) if bits == 4 else c.normal_()

        def step(q, k, v, caches, lens):
            lens.add_(1)
            q = tokens(prism_amd.qk_norm_rotary(heads(q), None, w, None, freqs, lens - 1))
            prism_amd.append_paged(k, v, *caches, table, lens, freqs=freqs)
            return prism_amd.flash_attn_paged(q, *caches, table, lens)

        eager, elens = [c.clone() for c in own], lens.clone()
        step(q, k, v, [c.clone() for c in own], lens.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(q, k, v, own, lens)
        for i in range(5):
            for t, s in ((q, 1), (k, 2), (v, 3)):
                t.copy_(randn(*t.shape, seed=100 * i + s))
            graph.replay()
            torch.cuda.synchronize()
            want = step(q, k, v, eager, elens)
            assert torch.equal(got, want) and torch.equal(lens, elens)
            assert all(torch.equal(a, b) for a, b in zip(own, eager))


def test_training_step_in_a_graph():
    """Forward and backward captured (work lists, cut lists and all), replayed with other
    inputs and other lengths: the bits of eager steps."""
    Hq, Hk, D = 4, 2, 64
    freqs, _ = prism_amd.rotary_frequencies(D)
    T = 1500
    bounds, at = cu([700, 500, 300]), places([700, 500, 300])
    args = [randn(T, H, D, seed=i) for i, H in enumerate((Hq, Hk, Hk))] + [torch.ones(D, device=DEV) for _ in "qk"]
    do = randn(T, Hq, D, seed=8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaves = [t.clone().requires_grad_(True) for t in args]

        def step():
            o = layer(*leaves, freqs, at, bounds)
            return [o.detach(), *torch.autograd.grad(o, leaves, do)]

        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
        for i, lens in enumerate(([700, 500, 300], [1500, 0, 0], [10, 1400, 90], [500, 500, 500])):
            for x, t in enumerate(leaves):
                t.data.copy_(randn(*t.shape, seed=50 + 10 * i + x))
            bounds.copy_(cu(lens))
            at.copy_(places(lens))
            graph.replay()
            torch.cuda.synchronize()
            got_now = [t.clone() for t in got]
            assert all(torch.equal(a, b) for a, b in zip(got_now, step())), lens


def test_two_graphs_do_not_share_workspaces():
    lens = [900, 300]
    bounds = cu(lens)
    ins = [[randn(1200, H, 64, seed=10 * s + i) for i, H in enumerate((4, 2, 2))] for s in range(2)]
    want = [prism_amd.flash_attn_packed(*x, bounds) for x in ins]
    torch.cuda.synchronize()
    graphs, got = [], []
    for x in ins:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(prism_amd.flash_attn_packed(*x, bounds))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    """Calls on two streams, behind long queues of other work, with their own inputs."""
    freqs, _ = prism_amd.rotary_frequencies(64)
    table, pages = table_for([700, 90], 16)
    lens = ints([700, 90])
    work = randn(2048, 2048)

    def calls(seed):
        q, k, v = (randn(790, H, 64, seed=seed + i) for i, H in enumerate((4, 2, 2)))
        kc, vc = prism_amd.paged_cache(pages, 16, 2, 64, bits=4)
        prism_amd.append_paged(k, v, kc, vc, table, lens, cu_seqlens=cu([700, 90]), freqs=freqs)
        return [prism_amd.flash_attn_packed(q, k, v, cu([700, 90])), prism_amd.flash_attn_paged(q[:4], kc, vc, table, lens),
                *prism_amd.gather_paged(kc, vc, table, cu([700, 90]), 790, head_dim=64)]

    want = [calls(s) for s in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in want]
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                x = work
                for _ in range(10):
                    x = (x @ work).clamp(-1, 1)
                got.append(calls(i + 1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


# ------------------------------------------------------------------ transforms
def test_vmap_gives_the_bits_of_a_loop():
    freqs, _ = prism_amd.rotary_frequencies(64)
    bounds, at = cu([5, 20, 11]), places([5, 20, 11])
    q, k, w = randn(3, 36, 4, 64, seed=1), randn(36, 3, 2, 64, seed=2), randn(64, seed=3)
    runs = []
    for mapped in (True, False):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, w)]
        f = lambda q, k, w: layer(q, k, k, w, w, freqs, at, bounds)  # noqa: E731
        out = torch.vmap(f, in_dims=(0, 1, None))(*leaves) if mapped else \
            torch.stack([f(leaves[0][i], leaves[1][:, i], leaves[2]) for i in range(3)])
        runs.append([out, *torch.autograd.grad(out, leaves, randn(*out.shape, seed=9))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    table, pages = table_for([36], 16)
    kc, vc = prism_amd.paged_cache(pages, 16, 2, 64)
    prism_amd.append_paged(k[:, 0], k[:, 1], kc, vc, table, ints([36]))
    got = torch.vmap(lambda x: prism_amd.flash_attn_paged(x, kc, vc, table, ints([36])))(q[:, :2])
    assert torch.equal(got, torch.stack([prism_amd.flash_attn_paged(x, kc, vc, table, ints([36])) for x in q[:, :2]]))


def test_vmap_of_the_caches():
    """Reading under vmap is the loop's; writing is refused, and nothing is written."""
    table, pages = table_for([36, 20], 16)
    kc, vc = prism_amd.paged_cache(pages, 16, 2, 64, bits=4)
    x = randn(56, 2, 64, seed=4)
    prism_amd.append_paged(x, x, kc, vc, table, ints([36, 20]), cu_seqlens=cu([36, 20]))
    read = lambda row: prism_amd.gather_paged(kc, vc, row[None], cu([20]), 22, head_dim=64)  # noqa: E731
    for a, b in zip(torch.vmap(read)(table), zip(*(read(row) for row in table))):
        assert torch.equal(a, torch.stack(b))
    before = kc.clone()
    with pytest.raises(RuntimeError, match="paged_append"):
        torch.vmap(lambda y: prism_amd.append_paged(y, y, kc, vc, table[:1], ints([3])))(randn(2, 3, 2, 64, seed=5))
    assert torch.equal(kc, before)


def test_tangents_and_second_derivatives_are_refused():
    import torch.autograd.forward_ad as forward_ad
    freqs, _ = prism_amd.rotary_frequencies(64)
    q, bounds, at = randn(9, 2, 64), cu([9]), places([9])
    with forward_ad.dual_level():
        d = forward_ad.make_dual(q, q)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            prism_amd.flash_attn_packed(d, q, q, bounds)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            prism_amd.qk_norm_rotary(heads(d), None, None, None, freqs, at)
        table, pages = table_for([9], 16)
        kc, vc = prism_amd.paged_cache(pages, 16, 2, 64)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            prism_amd.flash_attn_paged(d[:1], kc, vc, table, ints([9]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            prism_amd.append_paged(d, q, kc, vc, table, ints([9]))
    for f in (lambda t: prism_amd.flash_attn_packed(t, t, t, bounds),
              lambda t: prism_amd.qk_norm_rotary(heads(t), None, None, None, freqs, at)):
        t = q.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(t).float().pow(2).sum(), t, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            g.float().sum().backward()


def test_compiled_programs():
    """A training step compiled once with dynamic lengths, and a decoding step (whose
    append changes the caches): the eager bits."""
    torch._dynamo.reset()
    freqs, _ = prism_amd.rotary_frequencies(64)
    fast = torch.compile(layer, backend="aot_eager", dynamic=True, fullgraph=True)
    for n in (70, 71, 333, 1300):
        args = [randn(n, H, 64, seed=n + i) for i, H in enumerate((4, 2, 2))] + [randn(64, seed=5), randn(64, seed=6)]
        runs = []
        for f in (layer, fast):
            leaves = [t.clone().requires_grad_(True) for t in args]
            with torch.compiler.set_stance("default" if n == 70 else "fail_on_recompile"):
                o = f(*leaves, freqs, torch.arange(n, device=DEV), cu([n - 9, 9]))
            runs.append([o.detach(), *torch.autograd.grad(o, leaves, randn(*o.shape, seed=5))])
        assert all(torch.equal(a, b) for a, b in zip(*runs)), n

    table, pages = table_for([50, 20], 16)

    def step(q, k, v, kc, vc, lens):
        prism_amd.append_paged(k, v, kc, vc, table, lens, freqs=freqs)
        return prism_amd.flash_attn_paged(q, kc, vc, table, lens)

    for bits in (16, 4):
        caches = [[c.clone() for c in prism_amd.paged_cache(pages, 16, 2, 64, bits=bits)] for _ in "ab"]
        quick = torch.compile(step, backend="aot_eager", fullgraph=True)
        for i in range(3):
            q, k, v = (randn(2, H, 64, seed=i * 5 + x) for x, H in enumerate((4, 2, 2)))
            lens = ints([40 + i, 10 + i])
            assert torch.equal(step(q, k, v, *caches[0], lens), quick(q, k, v, *caches[1], lens))
            assert all(torch.equal(a, b) for a, b in zip(*caches))


def test_opcheck():
    freqs, _ = prism_amd.rotary_frequencies(64)
    at, bounds = torch.arange(12, device=DEV), cu([5, 7])
    q, k = randn(1, 4, 12, 64, seed=1), randn(1, 12, 2, 64, seed=2).transpose(1, 2)
    w = randn(64, seed=3)
    table, pages = table_for([5, 7], 16)
    lens = ints([5, 7])

    def run(op, *args):
        print("[case] opcheck", op, flush=True)
        torch.library.opcheck(getattr(torch.ops.prism, op).default, args, test_utils=("test_schema", "test_faketensor"))

    for kk, ww in ((k, w), (None, None)):
        run("qk_norm_rotary", q, kk, w, ww, 1e-6, freqs, at, [], True, 1.0)
        run("qk_norm_rotary_bwd", q, kk, q, kk, w, ww, 1e-6, freqs, at, [], True, 1.0, True, ww is not None)
    p, r = tokens(q), tokens(k)
    for flags in ((False, False), (True, True)):
        run("packed_fwd", p, r, r, bounds, bounds, True, 0.125, *flags)
    o, lse, rest = torch.ops.prism.packed_fwd(p, r, r, bounds, bounds, True, 0.125, True, True)
    run("packed_bwd", o, p, r, r, o, rest, lse, bounds, bounds, True, 0.125)
    for bits in (16, 4):
        kc, vc = prism_amd.paged_cache(pages, 16, 2, 64, bits=bits)
        run("paged_append", r, r, kc, vc, table, lens, bounds, freqs, None, [], True, 1.0)
        run("paged_gather", kc, vc, table, bounds, 12, 2, 64, False)
        run("paged_fwd", p[:2], kc, vc, table, lens, 2, 0.125, True)


def test_the_caches_version_counts():
    """torch knows that append_paged changed the caches."""
    table, pages = table_for([4], 16)
    kc, vc = prism_amd.paged_cache(pages, 16, 2, 64)
    before = kc._version, vc._version
    prism_amd.append_paged(randn(4, 2, 64), randn(4, 2, 64), kc, vc, table, ints([4]))
    assert kc._version > before[0] and vc._version > before[1]
    with torch.inference_mode():
        kc, vc = prism_amd.paged_cache(pages, 16, 2, 64)
        prism_amd.append_paged(randn(4, 2, 64), randn(4, 2, 64), kc, vc, table, ints([4]))
    prism_amd.append_paged(randn(4, 2, 64), randn(4, 2, 64), kc, vc, table, ints([4]))


def test_kernel_timing_sees_the_launches():
    from prism_amd import ops
    freqs, _ = prism_amd.rotary_frequencies(64)
    bounds, at = cu([30, 40]), places([30, 40])
    args = [randn(70, H, 64, seed=i) for i, H in enumerate((4, 2, 2))] + [randn(64, seed=5), randn(64, seed=6)]
    table, pages = table_for([30, 40], 16)
    kc, vc = prism_amd.paged_cache(pages, 16, 2, 64)
    with ops.kernel_timing() as tm:
        leaves = [t.clone().requires_grad_(True) for t in args]
        o = layer(*leaves, freqs, at, bounds)
        torch.autograd.grad(o, leaves, torch.ones_like(o))
        prism_amd.append_paged(args[1], args[2], kc, vc, table, ints([30, 40]), cu_seqlens=bounds)
        prism_amd.flash_attn_paged(args[0][:2], kc, vc, table, ints([30, 40]))
        prism_amd.gather_paged(kc, vc, table, bounds, 70)
    torch.cuda.synchronize()
    calls = {name: n for name, (n, ms) in ops.summarize(tm).items() if ms > 0}
    assert calls == {"prism_" + n: 1 for n in ("qk_norm_rotary", "qk_norm_rotary_bwd", "packed_fwd", "packed_bwd", "paged_append",
                                               "paged_fwd", "paged_gather")}


# ------------------------------------------------------------------ sizes
def test_offsets_past_32_bits():
    """Packed tensors of more than 2^31 elements and caches of more than 4 GB: the last
    sequence gives what it gives alone."""
    H, D, n, B = 8, 128, 500, 4500
    T = n * B  # 2.3e9 elements
    q = torch.zeros(T, H, D, device=DEV, dtype=torch.bfloat16)
    bounds = torch.arange(B + 1, device=DEV, dtype=torch.int32) * n
    for b in (0, B - 1):
        q[b * n:b * n + n] = randn(n, H, D, seed=b)
    leaf = q.requires_grad_(True)
    o = prism_amd.flash_attn_packed(leaf, leaf, leaf, bounds)
    (dq,) = torch.autograd.grad(o, leaf, o.detach())
    for b in (0, B - 1):
        one = q.detach()[b * n:b * n + n].clone().requires_grad_(True)
        want = prism_amd.flash_attn_packed(one, one, one, ints([0, n]))
        (dw,) = torch.autograd.grad(want, one, want.detach())
        for x, y in ((o.detach()[b * n:b * n + n], want.detach()), (dq[b * n:b * n + n], dw)):
            # (a launch of other sizes cuts the lists otherwise: sums in another order, rounded alike)
            assert (x.float() - y.float()).norm() <= 2.0 ** -8 * y.float().norm()
    del o, dq, leaf, q
    page = 64
    for bits, pages in ((16, 40000), (4, 140000)):
        kc, vc = prism_amd.paged_cache(pages, page, H, D, bits=bits)
        assert kc.numel() * kc.element_size() > 1 << 32
        k, v, x = randn(300, H, D, seed=1), randn(300, H, D, seed=2), randn(1, 16, D, seed=3)
        small = prism_amd.paged_cache(5, page, H, D, bits=bits)
        far, near = ints([[pages - 1, 3, pages - 7, pages // 2, pages - 2]]), ints([[0, 1, 2, 3, 4]])
        for caches, table in (((kc, vc), far), (small, near)):
            prism_amd.append_paged(k, v, *caches, table, ints([300]))
        assert torch.equal(kc[far[0].long()], small[0][near[0].long()])
        assert torch.equal(prism_amd.flash_attn_paged(x, kc, vc, far, ints([300])), prism_amd.flash_attn_paged(x, *small, near, ints([300])))
        a, b = (prism_amd.gather_paged(*c, t, ints([0, 300]), 300, head_dim=D) for c, t in (((kc, vc), far), (small, near)))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        del kc, vc


def test_many_short_sequences_and_one_long():
    """3,000 sequences of none to five tokens beside one of 2,000."""
    lens = [i % 6 for i in range(3000)] + [2000]
    T = sum(lens)
    q, k, v = (randn(T, H, 64, seed=i) for i, H in enumerate((4, 2, 2)))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = prism_amd.flash_attn_packed(*leaves, cu(lens))
    got = [o, *torch.autograd.grad(o, leaves, o.detach())]
    for b in (1, 5, 2999, 3000):
        s = slice(sum(lens[:b]), sum(lens[:b + 1]))
        one = [t.detach()[s].clone().requires_grad_(True) for t in (q, k, v)]
        w = prism_amd.flash_attn_packed(*one, ints([0, lens[b]]))
        want = [w, *torch.autograd.grad(w, one, o.detach()[s])]
        for x, y in zip(got, want):
            assert (x[s].float() - y.float()).norm() <= 2.0 ** -7 * y.float().norm()
    table, pages = table_for(lens[:3000], 16)
    kc, vc = prism_amd.paged_cache(pages, 16, 2, 64)
    head = sum(lens[:3000])
    with torch.no_grad():
        prism_amd.append_paged(k[:head], v[:head], kc, vc, table, ints(lens[:3000]), cu_seqlens=cu(lens[:3000]))
        gk, gv = prism_amd.gather_paged(kc, vc, table, cu(lens[:3000]), head)
    assert torch.equal(gk, k[:head]) and torch.equal(gv, v[:head])
