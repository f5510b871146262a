"""qk_norm_rotary against the formulas in float64: values and gradients over types,
layouts, head sizes (whole 16-byte pieces, half of them, single elements), parts of
heads and grids; its gradients against differences; bits that do not vary."""
import math

import pytest
import torch

import prism_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _turn(x, unit, inter):
    """float64 [B, H, S, D] times unit [B or 1, 1, S, R/2], pair by pair."""
    R = 2 * unit.shape[-1]
    rot = x[..., :R]
    pair = rot.unflatten(-1, (R // 2, 2)) if inter else rot.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit)
    return torch.cat([z.flatten(-2) if inter else z.transpose(-1, -2).flatten(-2), x[..., R:]], -1)


def _pairs(x, unit, inter):
    """The sizes of x's pairs, times the amplitude, in both of their channels."""
    one = torch.ones_like(unit)
    other = _turn(x, 1j * one, inter)  # (b in a's place, up to the sign)
    R = 2 * unit.shape[-1]
    return torch.cat([torch.hypot(x, other)[..., :R] * unit.abs().max(), x[..., R:]], -1)


def _oracle(x, w, unit, inter, eps, dy=None):
    x, w = x.double(), torch.ones(x.shape[-1], dtype=torch.float64, device=DEV) if w is None else w.double()
    inv = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    y = _turn(x * inv * w, unit, inter)
    if dy is None:
        return y, None, None
    g = _turn(dy.double(), unit.conj(), inter)
    dx = inv * (g * w - x * inv * (g * w * x * inv).mean(-1, keepdim=True))
    return y, dx, (g * x * inv).sum((0, 1, 2))


def _near(got, want, dtype, terms):
    """Half a step of the type, and for the fp32 arithmetic in between (sums of
    `terms` products, a square root, two rotations) 16 + terms/8 steps of 2^-24 of
    the largest value near: sums in any order are off by less than terms steps, and
    by their root when the signs vary."""
    scale = want.abs().amax(-1, keepdim=True).clamp(min=1e-30)
    bound = want.abs() * STEP[dtype] * (1 + 1e-3) + scale * 2.0 ** -24 * (16 + terms / 8)
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25  # (half a step below the normal range)
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1, f"{worst:.3f} of the bound"


CASES = [
    # B, Hq, Hk, S, D, R, interleaved, dtype, layout, sections
    (1, 1, 1, 1, 128, 128, True, torch.bfloat16, "bhsd", None),
    (3, 8, 2, 33, 128, 128, False, torch.bfloat16, "bshd", None),
    (2, 5, 5, 70, 64, 32, False, torch.float16, "bshd", None),
    (1, 4, 4, 24, 128, 128, True, torch.bfloat16, "bshd", (44, 42, 42)),
    (2, 3, 1, 19, 80, 80, False, torch.bfloat16, "bhsd", None),
    (2, 3, 1, 19, 80, 40, False, torch.bfloat16, "bhsd", None),    # halves of a piece
    (2, 3, 1, 19, 80, 20, False, torch.float32, "bhsd", None),     # single elements
    (1, 2, 2, 9, 256, 256, False, torch.float32, "bhsd", None),
    (1, 2, 2, 9, 256, 128, True, torch.bfloat16, "bhsd", None),
    (2, 2, 1, 7, 10, 6, True, torch.float16, "bhsd", None),
    (1, 2, 2, 5, 33, 2, False, torch.float32, "odd", None),
    (1, 4, 2, 12, 128, 128, True, torch.bfloat16, "odd", None),    # rows that are not 16-byte aligned
    (1, 4, 2, 12, 64, 64, False, torch.bfloat16, "columns", None),  # channels apart
    (1, 64, 8, 700, 32, 32, False, torch.bfloat16, "bshd", None),
]


def _make(g, B, H, S, D, dtype, layout):
    if layout == "bshd":
        return torch.randn(B, S, H, D, generator=g, device=DEV).to(dtype).transpose(1, 2)
    if layout == "odd":
        return torch.randn(B, H, S, D + 3, generator=g, device=DEV).to(dtype)[..., 1:D + 1]
    if layout == "columns":
        return torch.randn(B, H, D, S, generator=g, device=DEV).to(dtype).transpose(2, 3)
    return torch.randn(B, H, S, D, generator=g, device=DEV).to(dtype)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("weights", ["own", "fp32", "none"])
def test_against_float64(case, weights):
    B, Hq, Hk, S, D, R, inter, dtype, layout, sections = case
    g = torch.Generator(device=DEV).manual_seed(B * 1000 + S)
    q, k, dq, dk = (_make(g, B, H, S, D, dtype, layout) for H in (Hq, Hk, Hq, Hk))
    q[0, 0, 0] *= 100
    w = [None, None]
    if weights != "none":
        w = [(torch.rand(D, generator=g, device=DEV) + 0.5).to(dtype if weights == "own" else torch.float32) for _ in "qk"]
    freqs, _ = prism_amd.rotary_frequencies(R, sections=sections, device=DEV)
    if sections:
        pos = prism_amd.grid_positions((2, 3, 4))
        angle = torch.cat([pos.double()[:, a:a + 1] * f for a, f in enumerate(freqs.split([n // 2 for n in sections]))], -1)
    else:
        pos = torch.randint(0, 200000, (B, S), generator=g, device=DEV)
        angle = pos.double()[..., None] * freqs
    amp = 1.25
    unit = torch.polar(torch.full_like(angle, amp), angle).view(-1, 1, S, R // 2)
    kw = dict(eps=1e-5, interleaved=inter, sections=sections, amplitude=amp)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, *w) if t is not None]
    wl = leaves[2:] if weights != "none" else [None, None]
    oq, ok = prism_amd.qk_norm_rotary(leaves[0], leaves[1], *wl, freqs, pos, **kw)
    grads = torch.autograd.grad((oq, ok), leaves, (dq, dk))
    if layout in ("bhsd", "bshd"):
        assert oq.stride() == q.stride() and grads[0].stride() == q.stride()
    for i, (x, weight, dy, got) in enumerate(((q, w[0], dq, oq), (k, w[1], dk, ok))):
        y, dx, dw = _oracle(x, weight, unit, inter, 1e-5, dy)
        _near(got, y, dtype, D)
        _near(grads[i], dx, dtype, 2 * D)
        if weights != "none":
            # (a sum over B H S rows: steps of 2^-24 of the sum of the magnitudes.  The
            # magnitude of a turned a cos - b sin is that of the pair, (a^2 + b^2)^1/2, however
            # far the two cancel: each product is rounded, and the sine and cosine are 3e-8 off)
            rows = B * x.shape[1] * S
            xn = x.double() * (x.double().pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
            size = (_pairs(dy.double(), unit, inter) * xn).abs().sum((0, 1, 2))
            bound = dw.abs() * STEP[weight.dtype] * (1 + 1e-3) + size * 2.0 ** -24 * (24 + D / 8 + min(rows, 1024) / 8)
            if weight.dtype == torch.float16:
                bound = bound + 2.0 ** -25
            worst = ((grads[2 + i].double() - dw).abs() / bound.clamp(min=1e-300)).max().item()
            assert worst <= 1, f"{worst:.3f} of the bound"
    # the same without gradients, alone, and every time
    with torch.no_grad():
        assert torch.equal(prism_amd.qk_norm_rotary(q, k, *w, freqs, pos, **kw)[1], ok)
        assert torch.equal(prism_amd.qk_norm_rotary(q, None, w[0], None, freqs, pos, **kw), oq)
    again = prism_amd.qk_norm_rotary(leaves[0], leaves[1], *wl, freqs, pos, **kw)
    for a, b in zip(grads, torch.autograd.grad(again, leaves, (dq, dk))):
        assert torch.equal(a, b)


def test_gradients_of_one_output():
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k = (torch.randn(2, H, 9, 64, generator=g, device=DEV, requires_grad=True) for H in (4, 2))
    w = [torch.rand(64, generator=g, device=DEV).requires_grad_(True) for _ in "qk"]
    freqs, _ = prism_amd.rotary_frequencies(64)
    at = torch.arange(9, device=DEV)
    leaves = (q, k, *w)
    oq, ok = prism_amd.qk_norm_rotary(*leaves, freqs, at)
    dy = torch.randn_like(ok)
    both = torch.autograd.grad((oq, ok), leaves, (torch.zeros_like(oq), dy))
    oq, ok = prism_amd.qk_norm_rotary(*leaves, freqs, at)
    one = torch.autograd.grad(ok, leaves, dy, allow_unused=True)
    assert one[0] is None and one[2] is None
    assert torch.equal(one[1], both[1]) and torch.allclose(one[3], both[3], rtol=1e-5, atol=1e-6)


def test_gradients_against_differences():
    g = torch.Generator(device=DEV).manual_seed(6)
    q = torch.randn(1, 2, 5, 32, generator=g, device=DEV)
    w = torch.rand(32, generator=g, device=DEV) + 0.5
    freqs, _ = prism_amd.rotary_frequencies(16)
    at = torch.arange(5, device=DEV)
    c = torch.randn(1, 2, 5, 32, generator=g, device=DEV, dtype=torch.float64)
    f = lambda x, y: (prism_amd.qk_norm_rotary(x, None, y, None, freqs, at).double() * c).sum()  # noqa: E731
    ql, wl = q.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dq, dw = torch.autograd.grad((prism_amd.qk_norm_rotary(ql, None, wl, None, freqs, at) * c.float()).sum(), (ql, wl))
    for base, d, arg in ((q, dq, 0), (w, dw, 1)):
        for _ in range(6):
            e = torch.randn(base.shape, generator=g, device=DEV)
            h = 2.0 ** -6
            a, b = ((q + s * h * e, w) if arg == 0 else (q, w + s * h * e) for s in (1, -1))
            diff = (f(*a) - f(*b)).item() / (2 * h)
            want = (d.double() * e.double()).sum().item()
            # (the difference's own error: fp32 results of up to 320 values of size 2 over 2 h, and h^2 of the third derivative)
            assert abs(diff - want) <= 320 ** 0.5 * 2 * 2.0 ** -23 / (2 * h) * 8 + 40 * h * h * max(1.0, abs(want))


def test_not_finite_stays_in_its_head():
    q = torch.randn(1, 3, 4, 128, device=DEV).bfloat16()
    q[0, 1, 2, 7] = float("nan")
    q[0, 2, 0, 100] = float("inf")
    freqs, _ = prism_amd.rotary_frequencies(128)
    for inter in (True, False):
        y = prism_amd.qk_norm_rotary(q, None, None, None, freqs, torch.arange(4, device=DEV), interleaved=inter)
        bad = torch.zeros(1, 3, 4, dtype=torch.bool, device=DEV)
        bad[0, 1, 2] = bad[0, 2, 0] = True
        assert torch.isfinite(y[~bad]).all() and not torch.isfinite(y[bad]).all(-1).any()


def test_empty():
    freqs, _ = prism_amd.rotary_frequencies(64)
    q = torch.empty(2, 4, 0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = prism_amd.qk_norm_rotary(q, None, w, None, freqs, torch.arange(0, device=DEV))
    dq, dw = torch.autograd.grad(y.sum(), (q, w))
    assert y.shape == q.shape and dq.shape == q.shape and not dw.any()


def test_eps_zero_row():
    """All zeros and eps 0: the formula's NaN, in that head alone."""
    q = torch.randn(1, 2, 3, 64, device=DEV)
    q[0, 1, 1] = 0
    freqs, _ = prism_amd.rotary_frequencies(64)
    y = prism_amd.qk_norm_rotary(q, None, None, None, freqs, torch.arange(3, device=DEV), eps=0.0)
    assert torch.isnan(y[0, 1, 1]).all() and torch.isfinite(y).sum() == 5 * 64
    y = prism_amd.qk_norm_rotary(q, None, None, None, freqs, torch.arange(3, device=DEV))
    assert (y[0, 1, 1] == 0).all()
