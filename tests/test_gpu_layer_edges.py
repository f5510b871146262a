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
