"""apply_rotary against float64 (a product of complex numbers), forward and
backward, in both layouts, on parts of the head, several axes and far positions.

Tolerance: the angle is reduced in float64 (off by less than 1e-9 turns up to
position 2^31), sine and cosine are off by at most 2.5e-7 (series 3e-8, the
fp32 argument 6e-8 * pi / 4, Horner's roundings), the two products and their sum
add 2 u of the pair's length: 4e-7 amplitude |(a, b)| in all, and half |out| of
the output's type (half a subnormal step, 2^-25 in float16, below its smallest
normal number).
"""
import math

import pytest
import torch

import prism_amd

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def turned(x, freqs, positions, interleaved, sections, amplitude, sign=1):
    """(exact, length of each channel's pair) in float64."""
    R, B, S = 2 * freqs.numel(), x.shape[0], x.shape[2]
    p = positions.double()
    if sections is None:
        angle = p[..., None] * freqs
    else:
        n = torch.tensor([s // 2 for s in sections], device=p.device)
        axis = torch.repeat_interleave(torch.arange(len(sections), device=p.device), n)
        angle = p[..., axis] * freqs
    angle = angle.expand(B, S, R // 2)[:, None] * sign
    y = x.double().clone()
    a = y[..., 0:R:2] if interleaved else y[..., :R // 2]
    b = y[..., 1:R:2] if interleaved else y[..., R // 2:R]
    z = torch.complex(a.contiguous(), b.contiguous()) * torch.polar(torch.full_like(angle, amplitude), angle)
    length = torch.zeros_like(y)
    size = torch.hypot(a, b) * amplitude
    for at, v in ((0, z.real), (1, z.imag)):
        where = slice(at, R, 2) if interleaved else slice(at * (R // 2), (at + 1) * (R // 2))
        y[..., where] = v
        length[..., where] = size
    return y, length


def check(got, x, freqs, positions, interleaved, sections, amplitude, sign=1):
    assert got.dtype == x.dtype and got.shape == x.shape
    want, length = turned(x, freqs, positions, interleaved, sections, amplitude, sign)
    R = 2 * freqs.numel()
    e = torch.finfo(x.dtype).eps / 2
    tol = e * want.abs() + 4e-7 * length + torch.finfo(x.dtype).smallest_normal * e
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))
    assert torch.equal(got[..., R:], x[..., R:])


CASES = [  # B, S, Hq, Hk, D, R, sections, far
    (1, 1, 1, 1, 2, 2, None, 0), (1, 1, 32, 8, 128, 128, None, 200000), (16, 1, 8, 8, 64, 32, None, 5),
    (2, 77, 6, 2, 80, 40, None, 1000), (3, 50, 3, 1, 96, 96, None, 2 ** 30), (2, 33, 2, 2, 80, 20, None, 0),
    (1, 120, 5, 5, 128, 128, (44, 42, 42), 0), (2, 24, 4, 4, 128, 128, (44, 42, 42), 0),
    (1, 60, 2, 1, 64, 48, (16, 16, 12, 4), 0), (2, 9, 7, 3, 15, 6, None, 3), (1, 301, 3, 3, 256, 256, None, 0),
    (1, 5, 2, 2, 256, 2, None, 0), (1, 2500, 2, 2, 64, 64, None, 7),
]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:6]))
def test_against_float64(case, interleaved):
    B, S, Hq, Hk, D, R, sections, far = case
    g = torch.Generator(device="cuda").manual_seed(S + D)
    for dt in DT.values():
        q = torch.randn(B, Hq, S, D, generator=g, device="cuda").to(dt)
        k = torch.randn(B, S, Hk, D, generator=g, device="cuda").to(dt).transpose(1, 2)  # as a projection leaves it
        freqs, _ = prism_amd.rotary_frequencies(R, sections=sections)
        shape = (B, S) if far else (S,)
        positions = torch.randint(-50, 1000, shape + ((len(sections),) if sections else ()), generator=g, device="cuda",
                                  dtype=torch.int64 if B > 1 else torch.int32) + far
        how = (interleaved, sections, 1.25)
        kw = dict(interleaved=interleaved, sections=sections, amplitude=1.25)
        a, b = q.clone().requires_grad_(True), k.detach().requires_grad_(True)
        oq, ok = prism_amd.apply_rotary(a, b, freqs, positions, **kw)
        assert ok.stride() == k.stride() or k.numel() <= D  # the layout is kept
        check(oq.detach(), q, freqs, positions, *how)
        check(ok.detach(), k, freqs, positions, *how)
        dq, dk = torch.randn_like(q), torch.randn_like(k)
        gq, gk = torch.autograd.grad((oq, ok), (a, b), (dq, dk))
        check(gq, dq, freqs, positions, *how, sign=-1)
        check(gk, dk, freqs, positions, *how, sign=-1)
        assert torch.equal(prism_amd.apply_rotary(q, None, freqs, positions, **kw), oq.detach())
        (only,) = torch.autograd.grad(prism_amd.apply_rotary(a, b, freqs, positions, **kw)[1].float().sum(), b)
        assert torch.isfinite(only).all()


def test_strides_and_alignment():
    """Odd offsets, rows inside wider ones, broadcast heads: the same values as
    on a contiguous copy."""
    base = torch.randn(2, 6, 40, 140, device="cuda", dtype=torch.bfloat16)
    freqs, _ = prism_amd.rotary_frequencies(64)
    positions = torch.arange(40, device="cuda")
    for x in (base[..., :128], base[..., 1:129], base[..., 4:132], base[:, ::2, :, 8:136], base[:, :1, :, :128].expand(2, 5, 40, 128),
              base.transpose(1, 2).transpose(1, 2)[..., 12:140], base[:, :, :, 0:128].transpose(-1, -2).contiguous().transpose(-1, -2)):
        for inter in (True, False):
            got = prism_amd.apply_rotary(x, None, freqs, positions, interleaved=inter)
            want = prism_amd.apply_rotary(x.clone(memory_format=torch.contiguous_format), None, freqs, positions,
                                          interleaved=inter)
            assert torch.equal(got, want)
            check(got, x, freqs, positions, inter, None, 1.0)


def test_relative_positions():
    """Scores of turned queries and keys depend on the distance alone."""
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(1, 1, 1, 128, generator=g, device="cuda").expand(1, 1, 200, 128)
    k = torch.randn(1, 1, 1, 128, generator=g, device="cuda").expand(1, 1, 200, 128)
    freqs, _ = prism_amd.rotary_frequencies(128)
    at = torch.arange(200, device="cuda") * 997
    oq = prism_amd.apply_rotary(q, None, freqs, at + 13, interleaved=False)
    ok = prism_amd.apply_rotary(k, None, freqs, at, interleaved=False)
    dots = (oq.double() * ok.double()).sum(-1)
    # 128 terms, each off by at most 2 * 4e-7 of the lengths
    assert float((dots - dots[..., :1]).abs().max()) <= 2 * 8e-7 * float(q[0, 0, 0].norm() * k[0, 0, 0].norm())


def test_grid_positions():
    p = prism_amd.grid_positions((3, 4, 5)).cpu()
    want = torch.tensor([(t, h, w) for t in range(3) for h in range(4) for w in range(5)], dtype=torch.int32)
    assert torch.equal(p, want)


def test_graph_and_streams():
    q, k = (torch.randn(4, h, 1, 128, device="cuda", dtype=torch.bfloat16) for h in (32, 8))
    freqs, amp = prism_amd.rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=8192)
    positions = torch.randint(0, 65536, (4, 1), device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = prism_amd.apply_rotary(q, k, freqs, positions, amplitude=amp)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(other, prism_amd.apply_rotary(q, k, freqs, positions, amplitude=amp)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = prism_amd.apply_rotary(q, k, freqs, positions, amplitude=amp)
    for _ in range(3):
        q.normal_()
        k.normal_()
        positions += 1
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, prism_amd.apply_rotary(q, k, freqs, positions, amplitude=amp)))


def test_empty():
    freqs, _ = prism_amd.rotary_frequencies(64)
    for shape in ((0, 2, 3, 64), (2, 2, 0, 64), (2, 0, 3, 64)):
        q = torch.empty(shape, device="cuda")
        positions = torch.arange(shape[2], device="cuda")
        assert prism_amd.apply_rotary(q, None, freqs, positions).shape == shape


def test_opcheck():
    q, k = torch.randn(2, 3, 7, 64, device="cuda"), torch.randn(2, 1, 7, 64, device="cuda")
    freqs, _ = prism_amd.rotary_frequencies(32)
    at = torch.arange(7, device="cuda")
    torch.library.opcheck(torch.ops.prism.rotary.default, (q, k, freqs, at, [], True, 1.0, False),
                          test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.prism.rotary.default, (q, None, freqs, torch.stack([at, at], 1), [10, 6], False, 1.0, True),
                          test_utils=("test_schema", "test_faketensor"))
