"""rms_norm and rms_norm_quant (residual addition, root-mean-square norm, 8-bit
output) against float64, forward and backward.

Tolerances, from the arithmetic (u = 2^-24, half = eps / 2 of the type):
  s = 1 / sqrt(mean(h^2) + eps) of up to 16,384 fp32 terms, each thread adding
  at most 64 of them, then 6 + 16 partial sums: relative error of the sum below
  90 u, of s below 46 u; with the rounding of h, the two products and the
  division 50 u.  Where the output has 16 bits its rounding adds half |y|, and
  below the smallest normal number (float16: 2^-14) half of a subnormal step,
  which is 2^-24 there whatever y: 2^-25 (float16; bfloat16 2^-134).
  scale: 50 u of max |y|, two divisions more.  A code is the nearest to y /
  scale up to 60 u: |code * scale - y| <= half |y| (e4m3, subnormals 2^-10
  scale) or scale / 2 (int8), plus 60 u.
  Gradients with a residual read the stored h, off by half |h|, so xh is too:
  |dx - exact| <= s (half |xh c| + |xh| half mean |g xh|) + half |dx| + 100 u of
  the terms' magnitudes; dw: half sum |dy xh| + half |dw| + 200 u sum |dy xh|.
"""
import pytest
import torch

import prism_amd

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half(dt):
    return torch.finfo(dt).eps / 2


def rounded(dt, v):
    """Half a step of dt at v."""
    return half(dt) * v.abs() + torch.finfo(dt).smallest_normal * half(dt)


def make(M, N, dt, residual=True, w32=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, r = rnd(M, N).to(dt), (3 * rnd(M, N)).to(dt)
    w = (1 + 0.3 * rnd(N)).to(torch.float32 if w32 else dt)
    return x, (r if residual else None), w


def exact(x, r, w, eps):
    h = x.double() if r is None else x.double() + r.double()
    s = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, s, h * s * (1.0 if w is None else w.double())


def check(got, want, tol, what):
    got = got.detach()
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


# every kernel shape: one, four and sixteen waves a row, whole and part vectors,
# odd widths (single elements), the smallest and the largest
SIZES = [(1, 1), (3, 2), (7, 8), (130, 64), (5, 200), (9, 333), (4, 512), (33, 1000), (2, 1024), (6, 1536), (3, 2048),
         (5, 4097), (4, 5120), (3, 8192), (2, 10001), (3, 12288), (2, 16383), (2, 16384), (1500, 96)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("M,N", SIZES)
def test_forward_and_gradients(M, N, dt):
    dt = DT[dt]
    for residual, w32 in ((True, False), (False, True)):
        x, r, w = make(M, N, dt, residual, w32, seed=M + N)
        eps = 1e-5
        leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
        out = prism_amd.rms_norm(x, w, residual=r, eps=eps)
        y, h = out if residual else (out, None)
        assert y.dtype == dt and y.shape == x.shape
        h64, s, y64 = exact(x.detach(), None if r is None else r.detach(), w.detach(), eps)
        check(y, y64, rounded(dt, y64) + 50 * U * y64.abs(), "y")
        if residual:
            check(h, h64, rounded(dt, h64), "h")
        g = torch.Generator(device="cuda").manual_seed(1)
        dy = torch.randn(M, N, generator=g, device="cuda").to(dt)
        dh = torch.randn(M, N, generator=g, device="cuda").to(dt)
        grads = torch.autograd.grad((y, h) if residual else (y,), leaves, (dy, dh) if residual else (dy,))
        xh, gg = h64 * s, dy.double() * w.detach().double()
        c = (gg * xh).mean(-1, keepdim=True)
        want = s * (gg - xh * c) + (dh.double() if residual else 0)
        eh = half(dt) if residual else 0.0
        m = (gg * xh).abs().mean(-1, keepdim=True)
        tol = s * eh * ((xh * c).abs() + xh.abs() * m) * 1.01 + rounded(dt, want) + \
            100 * U * (s * (gg.abs() + xh.abs() * m) + (dh.double().abs() if residual else 0))
        check(grads[0], want, tol, "dx")
        if residual:
            assert torch.equal(grads[0], grads[1])
        a = (dy.double() * xh).abs().sum(0)
        wd = (dy.double() * xh).sum(0)
        check(grads[-1], wd, eh * a * 1.01 + rounded(w.dtype, wd) + 200 * U * a, "dw")


@pytest.mark.parametrize("out", ["e4m3", "int8"])
@pytest.mark.parametrize("M,N,dt", [(1, 1, "fp32"), (4, 5120, "bf16"), (9, 77, "fp16"), (70, 512, "bf16"),
                                    (3, 1536, "fp32"), (2, 16384, "bf16"), (2, 10001, "bf16"), (5, 12288, "fp16")])
def test_8_bits(M, N, dt, out):
    dt = DT[dt]
    x, r, w = make(M, N, dt, seed=N)
    r[:, ::5] *= 20
    if M > 2:
        x[1], r[1] = 0, 0  # a row of zeros
    codes, scale, h = prism_amd.rms_norm_quant(x, w, residual=r, eps=1e-6,
                                               out_dtype=torch.float8_e4m3fn if out == "e4m3" else torch.int8)
    h64, s, y64 = exact(x, r, w, 1e-6)
    qmax = 448.0 if out == "e4m3" else 127.0
    top = y64.abs().amax(-1)
    check(scale, (top / qmax).clamp(min=2.0 ** -126), 60 * U * top / qmax + 1e-45, "scale")
    check(h, h64, rounded(dt, h64), "h")
    back = codes.double() * scale.double()[:, None]
    sc = scale.double()[:, None]
    step = y64.abs() * 2.0 ** -4 + sc * 2.0 ** -10 if out == "e4m3" else sc * 0.5
    check(back, y64, step + 120 * U * (y64.abs() + sc), "value")
    if M > 2:
        assert (codes[1].float() == 0).all() and float(scale[1]) == 2.0 ** -126


def test_strides_and_views():
    """Rows inside a wider tensor, a leading slice, an odd offset, a transposed
    view, broadcast rows and weights (rows that are not aligned are added in
    another order than aligned ones, so only the bound is compared)."""
    torch.manual_seed(11)
    base = torch.randn(6, 40, 300, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(256, device="cuda", dtype=torch.bfloat16)
    views = [(base[:, :, :256], w), (base[:, :, 3:260], base[0, 0, :257]), (base[::2, 1:, 8:264], w),
             (base.transpose(1, 2)[:, :40], base[0, 0, :40]), (base[:1, :1, :256].expand(5, 3, 256), w)]
    for x, wv in views:
        y = prism_amd.rms_norm(x, wv)
        y64 = exact(x, None, wv, 1e-6)[2]
        check(y, y64, rounded(x.dtype, y64) + 50 * U * y64.abs(), "y")


def test_gradients_by_differences():
    """Directional derivative of a weighted sum of y and h in float32."""
    x, r, w = make(5, 768, torch.float32, seed=3)
    g = torch.Generator(device="cuda").manual_seed(9)
    a, b, vx, vr = (torch.randn(5, 768, generator=g, device="cuda") for _ in range(4))
    vw = torch.randn(768, generator=g, device="cuda")

    def loss(e):
        y, h = prism_amd.rms_norm(x + e * vx, w + e * vw, residual=r + e * vr)
        return float((y.double() * a.double()).sum() + (h.double() * b.double()).sum())

    e = 2.0 ** -6
    diff = (loss(e) - loss(-e)) / (2 * e)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, h = prism_amd.rms_norm(leaves[0], leaves[2], residual=leaves[1])
    dx, dr, dw = torch.autograd.grad((y, h), leaves, (a, b))
    want = float((dx.double() * vx.double()).sum() + (dr.double() * vr.double()).sum() + (dw.double() * vw.double()).sum())
    # truncation e^2 / 6 times third derivatives of about 1 per term (3,840
    # terms, random signs: sqrt(3840) ~ 62), rounding 3,840 * 2 u * 3 / (2 e)
    assert abs(diff - want) <= 62 * e * e * 4 + 3840 * 4 * U * 3 / (2 * e), (diff, want)


def test_partial_gradients_and_no_alias():
    x, r, w = make(6, 512, torch.bfloat16, seed=4)
    a = x.clone().requires_grad_(True)
    y, h = prism_amd.rms_norm(a, w, residual=r)
    (dx,) = torch.autograd.grad(h.float().sum(), a, retain_graph=True)  # only the residual stream goes on
    assert torch.equal(dx, torch.ones_like(dx))
    (dy_only,) = torch.autograd.grad(y.float().sum(), a)
    assert torch.isfinite(dy_only).all()
    wl = w.clone().requires_grad_(True)  # the weight alone
    (dw,) = torch.autograd.grad(prism_amd.rms_norm(x, wl).float().sum(), wl)
    assert dw.shape == w.shape
    rl = r.clone().requires_grad_(True)
    a.grad = None
    y, h = prism_amd.rms_norm(a, w, residual=rl)
    (y.float().sum() + h.float().sum()).backward()
    assert torch.equal(a.grad, rl.grad) and a.grad.data_ptr() != rl.grad.data_ptr()


def test_empty_and_not_finite():
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x = torch.empty(0, 3, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = prism_amd.rms_norm(x, w)
    assert y.shape == x.shape
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert dx.shape == x.shape and (dw == 0).all()
    codes, scale = prism_amd.rms_norm_quant(x.detach(), w.detach())
    assert codes.shape == x.shape and scale.shape == x.shape[:-1]
    x = torch.randn(4, 64, device="cuda", dtype=torch.bfloat16)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    y = prism_amd.rms_norm(x, w.detach())
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()  # rows stay apart
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 7])
    codes, scale = prism_amd.rms_norm_quant(x, w.detach())
    assert torch.isfinite(scale[[0, 3]]).all() and not torch.isfinite(scale[[1, 2]]).any()


def test_graph_and_streams():
    x, r, w = make(37, 1536, torch.bfloat16, seed=6)
    eager = prism_amd.rms_norm_quant(x, w, residual=r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = prism_amd.rms_norm_quant(x, w, residual=r)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = prism_amd.rms_norm_quant(x, w, residual=r)
        y = prism_amd.rms_norm(x, w)
    for seed in (7, 8, 9):
        nx, nr, _ = make(37, 1536, torch.bfloat16, seed=seed)
        x.copy_(nx)
        r.copy_(nr)
        graph.replay()
        torch.cuda.synchronize()
        want = prism_amd.rms_norm_quant(x, w, residual=r)
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
        assert torch.equal(y, prism_amd.rms_norm(x, w))


def test_backward_captured():
    x, r, w = make(300, 768, torch.float32, seed=6)
    dy = torch.randn(300, 768, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]

    def step():
        y, h = prism_amd.rms_norm(leaves[0], leaves[2], residual=leaves[1])
        return torch.autograd.grad((y, h), leaves, (dy, dy))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2, 3):
        with torch.no_grad():
            for t, n in zip(leaves, make(300, 768, torch.float32, seed=seed)):
                t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_opcheck():
    x, r, w = make(5, 96, torch.bfloat16)
    for args in ((x, r, w, 1e-6, 1, True), (x, None, w.float(), 1e-6, 3, False), (x, r, None, 1e-6, 4, True)):
        torch.library.opcheck(torch.ops.prism.rms_norm.default, args, test_utils=("test_schema", "test_faketensor"))
    inv = torch.ones(5, device="cuda")
    for dh, want in ((r, True), (None, False)):
        torch.library.opcheck(torch.ops.prism.rms_norm_bwd.default, (x, dh, r, w, inv, want),
                              test_utils=("test_schema", "test_faketensor"))


def test_second_derivatives_are_refused_and_changed_inputs_seen():
    x, r, w = (t.requires_grad_(True) for t in make(4, 64, torch.float32))
    freqs, _ = prism_amd.rotary_frequencies(64)
    at = torch.arange(5, device="cuda")
    q = torch.randn(1, 2, 5, 64, device="cuda").half().requires_grad_(True)
    for y, leaf in ((prism_amd.rms_norm(x, w, residual=r)[0], x),
                    (prism_amd.apply_rotary(q, None, freqs, at), q), (prism_amd.flash_attn_window(q, q, q, 2), q)):
        (g,) = torch.autograd.grad(y.float().sum(), leaf, create_graph=True)
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="differentiated again"):
            g.float().sum().backward()
    y, h = prism_amd.rms_norm(x, w, residual=r)
    h.data.mul_(1)  # (not seen: .data has no version)
    with torch.no_grad():
        h.add_(1)   # what the backward reads has changed
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
