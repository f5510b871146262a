"""Timed cases of the operators around the attention: what a transformer layer
runs between its residual stream and its attention's output.

  norm     rms_norm / rms_norm_quant: residual addition and root-mean-square
           norm, output in the input's type or in 8 bits with a scale per row
  rotary   apply_rotary: rotary positions on queries and keys
  window   flash_attn_window: attention over a sliding window and the first
           tokens (sinks): prompts, training steps, single tokens over a cache

``listed`` holds the named cases, ``draw`` makes others of the same ranges,
``prepare`` makes a case's inputs, ``run`` makes one pass (where ``own`` is
false in plain torch operations, 32 bits, rounded once at the end; where it is
true through the framework's entry points), ``work`` counts what a pass cannot
do without and ``exact`` computes it in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
QMAX = {"e4m3": 448.0, "int8": 127.0}
TINY = 2.0 ** -126


# ------------------------------------------------------------------ cases
def _norm(rows, width, *, dtype="bf16", residual=True, out="same", train=False, name=None):
    c = dict(op="norm", rows=rows, width=width, dtype=dtype, residual=residual, out=out, train=train)
    return dict(c, name=name) if name else c


def _rotary(B, S, Hq, Hk, D, *, rotary_dim=None, interleaved=True, axes="", scaling="none", far=0, dtype="bf16",
            projected=False, train=False, name=None):
    """axes: "" for one position a token, else "TxHxW" (S tokens of that grid,
    three positions a token); far: the first position; projected: the tensors
    are [B, S, H, D] in memory, as a projection leaves them."""
    c = dict(op="rotary", B=B, S=S, Hq=Hq, Hk=Hk, D=D, rotary_dim=rotary_dim or D, interleaved=interleaved, axes=axes,
             scaling=scaling, far=far, dtype=dtype, projected=projected, train=train)
    return dict(c, name=name) if name else c


def _window(B, Sq, Sk, Hq, Hk, D, window, sinks, *, causal=True, ragged=False, dtype="bf16", projected=False,
            train=False, name=None):
    """ragged: the sequences' lengths differ (queries and keys alike where
    Sq == Sk: rows padded on the right; keys alone in a cache)."""
    c = dict(op="window", B=B, Sq=Sq, Sk=Sk, Hq=Hq, Hk=Hk, D=D, window=window, sinks=sinks, causal=causal,
             ragged=ragged, dtype=dtype, projected=projected, train=train)
    return dict(c, name=name) if name else c


def listed():
    return [
        # Four new tokens of a stream through a layer's norm before 8-bit
        # projections: latency.
        _norm(4, 5120, out="e4m3", name="norm_token_e4m3"),
        # A 720p clip (21 x 45 x 80 latent tokens) of the same layer: the
        # largest, bandwidth.
        _norm(75600, 5120, out="e4m3", name="norm_720p_e4m3"),
        # A training step of a short 480p clip (9 x 30 x 52).
        _norm(14040, 5120, train=True, name="norm_480p_train"),
        # The audio tower's 2,000 tokens in float32, no residual, training.
        _norm(2000, 1536, dtype="fp32", residual=False, train=True, name="norm_audio_train"),
        # One new token of each of 16 streams, far beyond the trained length.
        _rotary(16, 1, 32, 8, 128, interleaved=False, scaling="yarn", far=200000, name="rotary_token"),
        # Queries and keys of a 720p clip, 40 heads, as the projections leave
        # them, three axes, inference.
        _rotary(1, 75600, 40, 40, 128, axes="21x45x80", projected=True, name="rotary_720p"),
        # A text or audio batch in training: part of a small head, float32,
        # an odd length.
        _rotary(2, 4999, 16, 4, 64, rotary_dim=32, interleaved=False, scaling="linear", dtype="fp32", train=True,
                name="rotary_part_train"),
        # One new token of each of eight streams of different lengths over a
        # cache with room for 32,768: window and sinks.
        _window(8, 1, 32768, 32, 8, 128, 4096, 4, ragged=True, name="window_token"),
        # Two long streams over caches laid out by token, a wide window.
        _window(2, 1, 262144, 32, 8, 128, 131072, 64, dtype="fp16", projected=True, name="window_token_long"),
        # A prompt of odd length, shared key heads.
        _window(1, 16001, 16001, 32, 8, 128, 4096, 16, name="window_prompt"),
        # A training step over right-padded sequences, small heads.
        _window(2, 4096, 4096, 16, 4, 64, 1024, 4, ragged=True, dtype="fp16", train=True, name="window_train"),
        # A training step over a 480p clip's tokens, one GPU's heads: three
        # latent frames (of 30 x 52) to both sides, the first frame always
        # visible.
        _window(1, 14040, 14040, 5, 5, 128, 4680, 1560, causal=False, train=True, name="window_480p_train"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "window", "window"])
    train = rng.random() < 0.45
    if op == "norm":
        out = "same" if train else rng.choice(["same", "e4m3", "e4m3", "int8"])
        dtype = rng.choice(["bf16", "bf16", "fp16"] if out == "int8" else ["bf16", "bf16", "fp16", "fp32"])
        width = _log(rng, 8, 16384)
        if rng.random() < 0.6:
            width = max(8, width // 64 * 64)
        rows = _log(rng, 1, min(60000, 12e7 / width))
        return _norm(rows, width, dtype=dtype, residual=rng.random() < 0.6, out=out, train=train)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    Hk = rng.choice([1, 2, 4, 5, 8])
    Hq = Hk * rng.choice([1, 1, 2, 3, 4, 8])
    B = rng.choice([1, 1, 2, 3, 5, 8])
    if op == "rotary":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        D = rng.choice([32, 64, 64, 80, 128, 128, 128, 256])
        part = rng.choice([D, D, D, D // 2, D // 4])
        axes, S = "", _log(rng, 1, min(40000, 2.5e8 / (B * Hq * D)))
        if rng.random() < 0.35:
            T, H, W = rng.randint(1, 13), rng.randint(3, 45), rng.randint(4, 60)
            axes, S, part, B = "%dx%dx%d" % (T, H, W), T * H * W, D, 1
        return _rotary(B, S, Hq, Hk, D, rotary_dim=part, interleaved=rng.random() < 0.5, axes=axes,
                       scaling="none" if axes else rng.choice(["none", "linear", "ntk", "yarn"]),
                       far=0 if axes else rng.choice([0, 0, 777, 300000]), dtype=dtype,
                       projected=rng.random() < 0.5, train=train)
    D = rng.choice([64, 128, 128])
    if not train and rng.random() < 0.5:  # new tokens over a cache
        Sq, Sk = rng.choice([1, 1, 1, 2, 5]), _log(rng, 1, 120000)
        W = min(_log(rng, 16, 40000), 2 * Sk)
        return _window(B, min(Sq, Sk), Sk, Hq, Hk, D, W, rng.choice([0, 1, 4, 64, 100]), ragged=rng.random() < 0.7,
                       dtype=dtype, projected=rng.random() < 0.5)
    S = _log(rng, 2, max(64, min(9000, math.sqrt(1.5e9 / (B * Hq)))))
    W = min(_log(rng, 8, 6000), 2 * S)
    return _window(B, S, S, Hq, Hk, D, W, rng.choice([0, 1, 4, 70, 300]), causal=rng.random() < 0.7,
                   ragged=rng.random() < 0.4, dtype=dtype, projected=rng.random() < 0.5, train=train)


# ------------------------------------------------------------------ inputs
def _frequencies(c):
    """float64 angle per position of every pair, and the factor on the rotated
    channels (scalings: 8 times a trained length of 8,192)."""
    R, base, factor, trained = c["rotary_dim"], 10000.0, 8.0, 8192
    if c["axes"]:
        parts = _sections(R)
        return torch.cat([base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n) for n in parts]), 1.0
    i = torch.arange(0, R, 2, dtype=torch.float64)
    if c["scaling"] == "ntk":
        return (base * factor ** (R / (R - 2.0))) ** (-i / R), 1.0
    f = base ** (-i / R)
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] == "yarn":  # pairs that turn 32 times or more in the trained length stay, below once are divided
        low = R * math.log(trained / (32.0 * 2 * math.pi)) / (2 * math.log(base))
        high = R * math.log(trained / (1.0 * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(low), 0), min(math.ceil(high), R // 2 - 1)
        ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _sections(R):
    """Channels of the three axes of a video head: two sixths (rounded down to
    whole pairs) for height and width, the rest for time."""
    side = 2 * (R // 6)
    return [R - 2 * side, side, side]


def _heads(g, B, H, S, D, dtype, projected):
    """[B, H, S, D], in memory as such or as [B, S, H, D]."""
    if projected:
        return torch.randn(B, S, H, D, generator=g, device=DEVICE, dtype=dtype).transpose(1, 2)
    return torch.randn(B, H, S, D, generator=g, device=DEVICE, dtype=dtype)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "norm":
        M, N = c["rows"], c["width"]
        s["x"] = torch.randn(M, N, generator=g, device=DEVICE, dtype=dt)
        # a residual stream: larger than what a layer adds, a few channels far larger
        s["r"] = torch.randn(M, N, generator=g, device=DEVICE, dtype=dt).mul_(3) if c["residual"] else None
        if c["residual"]:
            s["r"][:, ::97] *= 10
        s["w"] = torch.rand(N, generator=g, device=DEVICE).add_(0.5).to(dt)
        if c["train"]:
            s["dy"] = torch.randn(M, N, generator=g, device=DEVICE, dtype=dt)
            s["dh"] = torch.randn(M, N, generator=g, device=DEVICE, dtype=dt) if c["residual"] else None
        return s
    if c["op"] == "rotary":
        B, S = c["B"], c["S"]
        s["q"] = _heads(g, B, c["Hq"], S, c["D"], dt, c["projected"])
        s["k"] = _heads(g, B, c["Hk"], S, c["D"], dt, c["projected"])
        f, s["amplitude"] = _frequencies(c)
        s["freqs"] = f.to(DEVICE)
        if c["axes"]:
            grid = [int(n) for n in c["axes"].split("x")]
            at = torch.meshgrid(*[torch.arange(n, device=DEVICE, dtype=torch.int32) for n in grid], indexing="ij")
            s["positions"] = torch.stack(at, -1).view(S, 3)
        else:  # every stream at a place of its own
            first = torch.randint(0, 1000, (B, 1), generator=g, device=DEVICE) + c["far"]
            s["positions"] = first + torch.arange(S, device=DEVICE)
        if c["train"]:
            s["dq"] = _heads(g, B, c["Hq"], S, c["D"], dt, c["projected"])
            s["dk"] = _heads(g, B, c["Hk"], S, c["D"], dt, c["projected"])
        return s
    B, Sq, Sk, D = c["B"], c["Sq"], c["Sk"], c["D"]
    s["q"] = _heads(g, B, c["Hq"], Sq, D, dt, c["projected"])
    s["k"] = _heads(g, B, c["Hk"], Sk, D, dt, c["projected"])
    s["v"] = _heads(g, B, c["Hk"], Sk, D, dt, c["projected"])
    s["q_lens"] = s["kv_lens"] = None
    if c["ragged"]:
        n = torch.randint(max(1, Sk // 2), Sk + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
        s["kv_lens"] = n
        s["q_lens"] = n.clone() if Sq == Sk else None
    if c["train"]:
        s["do"] = _heads(g, B, c["Hq"], Sq, D, dt, c["projected"])
    return s


# ------------------------------------------------------------------ one pass
def _plain_norm(c, s):
    dt, eps = DTYPES[c["dtype"]], 1e-6
    w = s["w"].float()
    h = s["x"].float()
    if c["residual"]:
        h = h + s["r"].float()
    inv = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    xh = h * inv
    y = xh * w
    out = {}
    if c["residual"]:
        out["h"] = h.to(dt)
    if c["out"] != "same":
        scale = (y.abs().amax(-1) / QMAX[c["out"]]).clamp(min=TINY)
        z = y / scale[:, None]
        out["scale"] = scale
        if c["out"] == "e4m3":
            out["q"] = z.to(torch.float8_e4m3fn)
        else:
            out["values"] = (z.round() * scale[:, None]).to(dt)
        return out
    out["y"] = y.to(dt)
    if c["train"]:
        dy = s["dy"].float()
        gy = dy * w
        dx = inv * (gy - xh * (gy * xh).mean(-1, keepdim=True))
        if c["residual"]:
            dx = dx + s["dh"].float()
            out["dr"] = dx.to(dt)
        out["dx"] = dx.to(dt)
        out["dw"] = (dy * xh).sum(0).to(dt)
    return out


def _own_norm(c, s):
    import prism_amd
    out = {}
    if c["out"] != "same":
        qt = torch.float8_e4m3fn if c["out"] == "e4m3" else torch.int8
        got = prism_amd.rms_norm_quant(s["x"], s["w"], residual=s["r"], eps=1e-6, out_dtype=qt)
        out["scale"] = got[1]
        if c["out"] == "e4m3":
            out["q"] = got[0]
        else:
            out["values"] = (got[0].float() * got[1][:, None]).to(s["x"].dtype)
        if c["residual"]:
            out["h"] = got[2]
        return out
    if not c["train"]:
        got = prism_amd.rms_norm(s["x"], s["w"], residual=s["r"], eps=1e-6)
        return {"y": got[0], "h": got[1]} if c["residual"] else {"y": got}
    x, w = (s[n].detach().requires_grad_(True) for n in ("x", "w"))
    if c["residual"]:
        r = s["r"].detach().requires_grad_(True)
        y, h = prism_amd.rms_norm(x, w, residual=r, eps=1e-6)
        dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (s["dy"], s["dh"]))
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dr": dr, "dw": dw}
    y = prism_amd.rms_norm(x, w, eps=1e-6)
    dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def _turn(c, x, cos, sin):
    """x [B, H, S, D] turned by the angles of cos, sin [.., S, R/2]."""
    R = c["rotary_dim"]
    rot, rest = x[..., :R].float(), x[..., R:]
    if c["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = rot[..., :R // 2], rot[..., R // 2:]
        rot = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([rot.to(x.dtype), rest], -1)


def _plain_rotary(c, s):
    p = s["positions"]
    if c["axes"]:
        n = torch.tensor([m // 2 for m in _sections(c["rotary_dim"])])
        axis = torch.repeat_interleave(torch.arange(3), n).to(DEVICE)
        angle = p.double()[:, axis] * s["freqs"]  # [S, R/2]
    else:
        angle = (p.double()[..., None] * s["freqs"])[:, None]  # [B, 1, S, R/2]
    cos, sin = (t.mul(s["amplitude"]).float() for t in (angle.cos(), angle.sin()))
    out = {"q": _turn(c, s["q"], cos, sin), "k": _turn(c, s["k"], cos, sin)}
    if c["train"]:
        out["dq"], out["dk"] = _turn(c, s["dq"], cos, -sin), _turn(c, s["dk"], cos, -sin)
    return out


def _own_rotary(c, s):
    import prism_amd
    kw = dict(interleaved=c["interleaved"], amplitude=s["amplitude"],
              sections=_sections(c["rotary_dim"]) if c["axes"] else None)
    if not c["train"]:
        q, k = prism_amd.apply_rotary(s["q"], s["k"], s["freqs"], s["positions"], **kw)
        return {"q": q, "k": k}
    q0, k0 = (s[n].detach().requires_grad_(True) for n in ("q", "k"))
    q, k = prism_amd.apply_rotary(q0, k0, s["freqs"], s["positions"], **kw)
    dq, dk = torch.autograd.grad((q, k), (q0, k0), (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _plain_window(c, s):
    B, Sq, Sk, Hq, Hk, D = (c[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D"))
    dt, G, scale = DTYPES[c["dtype"]], c["Hq"] // c["Hk"], 1.0 / math.sqrt(D)
    rows = lambda t: t.float().reshape(B, Hk, G * Sq, D)  # noqa: E731
    q, k, v = rows(s["q"]), s["k"].float().contiguous(), s["v"].float().contiguous()
    nk = s["kv_lens"].long()[:, None, None] if c["ragged"] else torch.full((B, 1, 1), Sk, device=DEVICE)
    nq = s["q_lens"].long()[:, None, None] if s["q_lens"] is not None else torch.full((B, 1, 1), Sq, device=DEVICE)
    i, j = torch.arange(Sq, device=DEVICE)[:, None], torch.arange(Sk, device=DEVICE)
    d = nk - nq + i - j  # [B, Sq, Sk]: how far the key is behind the query
    seen = ((d < c["window"]) | (j < c["sinks"])) & (d >= 0) if c["causal"] else \
        (d.abs() < c["window"]) | (j < c["sinks"])
    seen = (seen & (j < nk) & (i < nq))[:, None, None]
    x = (q @ k.transpose(-1, -2).contiguous()).mul_(scale).view(B, Hk, G, Sq, Sk).masked_fill_(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    e = x.sub_(top.masked_fill(torch.isinf(top), 0.0)).exp_()
    p = e.div_(e.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, Hk, G * Sq, Sk)
    o = p @ v
    out = {"o": o.view(B, Hq, Sq, D).to(dt)}
    if c["train"]:
        do = rows(s["do"])
        dv = p.transpose(-1, -2).contiguous() @ do
        ds = (do @ v.transpose(-1, -2).contiguous()).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"] = (ds @ k).view(B, Hq, Sq, D).to(dt)
        out["dk"], out["dv"] = (ds.transpose(-1, -2).contiguous() @ q).to(dt), dv.to(dt)
    return out


def _own_window(c, s):
    import prism_amd
    kw = dict(sinks=c["sinks"], causal=c["causal"], q_lens=s["q_lens"], kv_lens=s["kv_lens"])
    if not c["train"]:
        return {"o": prism_amd.flash_attn_window(s["q"], s["k"], s["v"], c["window"], **kw)}
    q, k, v = (s[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
    o = prism_amd.flash_attn_window(q, k, v, c["window"], **kw)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


_PLAIN = {"norm": _plain_norm, "rotary": _plain_rotary, "window": _plain_window}
_OWN = {"norm": _own_norm, "rotary": _own_rotary, "window": _own_window}


def run(state):
    c = state["case"]
    return (_OWN if own else _PLAIN)[c["op"]](c, state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Inputs read once and outputs written once; of a window's keys and
    values what its queries see (ragged lengths at their mean, three quarters),
    4 D operations a seen pair, 14 D with the backward."""
    c = case
    es = BYTES[c["dtype"]]
    if c["op"] == "norm":
        n, M = float(c["rows"]) * c["width"], c["rows"]
        r = 1 if c["residual"] else 0
        out = es if c["out"] == "same" else 1
        b = n * (es * (1 + 2 * r) + out) + es * c["width"] + (0 if c["out"] == "same" else 4 * M)
        if c["train"]:  # dy, dh, h (or x) read, dx, dr, dw written
            b += n * es * (3 + 2 * r) + es * c["width"]
        return {"bytes": float(b), "flops": n * (5 + r + (9 if c["train"] else 0))}
    if c["op"] == "rotary":
        n = float(c["B"]) * c["S"] * (c["Hq"] + c["Hk"]) * c["D"] * (2 if c["train"] else 1)
        return {"bytes": 2 * es * n + 8.0 * c["B"] * c["S"], "flops": 3 * n}
    B, Sq, Sk, Hq, Hk, D, W = (c[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D", "window"))
    nk = max(1.0, 0.75 * Sk if c["ragged"] else Sk)
    nq = nk if Sq == Sk else float(Sq)
    side = min(W, nk) if c["causal"] else min(2 * W - 1, nk)
    if Sq == Sk:  # a query near an end sees less
        span = min(W, nk)
        one = span - span * (span - 1) / (2 * nk)
        side = one if c["causal"] else min(2 * one - 1, nk)
        seen = min(nk, side + min(c["sinks"], nk) * (max(0.0, nk - side) / nk))
        kept = nk
    else:
        seen = kept = min(nk, side + c["sinks"] + Sq - 1)
    pairs = B * Hq * nq * max(1.0, seen)
    b = es * D * B * (2 * Hq * Sq + 2 * Hk * kept)
    if c["train"]:
        return {"bytes": float(b + es * D * B * (2 * Hq * Sq + 2 * Hk * Sk)), "flops": 14.0 * D * pairs}
    return {"bytes": float(b), "flops": 4.0 * D * pairs}


# ------------------------------------------------------------------ float64
def _exact_norm(c, s):
    res = {k: [] for k in ("y", "h", "scale", "q", "values", "dx")}
    dw = torch.zeros(c["width"], dtype=torch.float64, device=DEVICE)
    for a in range(0, c["rows"], 8192):
        part = slice(a, a + 8192)
        h = s["x"][part].to(torch.float64)
        if c["residual"]:
            h += s["r"][part]
            res["h"].append(h)
        length = (h.pow(2).sum(1) / c["width"] + 1e-6).sqrt()
        unit = h / length[:, None]
        y = unit * s["w"].double()
        if c["out"] != "same":
            scale = torch.clamp_min(y.abs().max(1).values / QMAX[c["out"]], TINY)
            res["scale"].append(scale)
            res["q" if c["out"] == "e4m3" else "values"].append(y / scale[:, None] if c["out"] == "e4m3" else y)
        else:
            res["y"].append(y)
        if c["train"]:
            gy = s["dy"][part].double()
            dw += (gy * unit).sum(0)
            gy = gy * s["w"].double()
            dx = (gy - unit * (unit * gy).sum(1, keepdim=True) / c["width"]) / length[:, None]
            res["dx"].append(dx + s["dh"][part] if c["residual"] else dx)
    out = {k: torch.cat(v) for k, v in res.items() if v}
    if c["train"]:
        out["dw"] = dw
        if c["residual"]:
            out["dr"] = out["dx"]
    return out


def _exact_rotary(c, s):
    """As a product of complex numbers."""
    R = c["rotary_dim"]
    p = s["positions"].double()
    if c["axes"]:
        n = [m // 2 for m in _sections(R)]
        parts = [p[:, a:a + 1] * f for a, f in enumerate(torch.split(s["freqs"], n))]
        unit = torch.polar(torch.tensor(1.0, dtype=torch.float64, device=DEVICE), torch.cat(parts, -1))[None]
    else:
        unit = torch.polar(torch.tensor(1.0, dtype=torch.float64, device=DEVICE), p[..., None] * s["freqs"])
    unit = unit * s["amplitude"]

    def turned(x, by):
        y = x.double()
        for h in range(x.shape[1]):
            z = y[:, h, :, :R]
            pair = z.unflatten(-1, (R // 2, 2)) if c["interleaved"] else z.unflatten(-1, (2, R // 2)).transpose(-1, -2)
            z2 = torch.view_as_real(torch.complex(pair[..., 0].contiguous(), pair[..., 1].contiguous()) * by)
            y[:, h, :, :R] = z2.flatten(-2) if c["interleaved"] else z2.transpose(-1, -2).flatten(-2)
        return y

    out = {"q": turned(s["q"], unit), "k": turned(s["k"], unit)}
    if c["train"]:
        out["dq"], out["dk"] = turned(s["dq"], unit.conj()), turned(s["dk"], unit.conj())
    return out


def _exact_window(c, s):
    """One sequence, one head and a run of queries at a time, over the keys
    that the run can see."""
    B, Sq, Sk, Hq, Hk, D, W = (c[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D", "window"))
    G, run_of = Hq // Hk, 2048
    o = torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device=DEVICE)
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(B, Hk, Sk, D, dtype=torch.float64, device=DEVICE) for _ in "kv")
    for b in range(B):
        nk = int(s["kv_lens"][b]) if c["ragged"] else Sk
        nq = int(s["q_lens"][b]) if s["q_lens"] is not None else Sq
        for a in range(0, nq, run_of):
            p = torch.arange(a, min(a + run_of, nq), device=DEVICE) + nk - nq
            first, last = int(p[0]) - W + 1, int(p[-1]) + (1 if c["causal"] else W)
            j = torch.arange(nk, device=DEVICE)
            j = j[((j >= first) | (j < c["sinks"])) & ((j < last) | (not c["causal"] and j < c["sinks"]))]
            gap = p[:, None] - j[None]
            hidden = ~((gap < W) & (gap > -W) | (j < c["sinks"])[None])
            if c["causal"]:
                hidden |= gap < 0
            empty = hidden.all(1, keepdim=True)
            for h in range(Hq):
                qh = s["q"][b, h, a:a + len(p)].double()
                kh, vh = s["k"][b, h // G, j].double(), s["v"][b, h // G, j].double()
                x = qh @ kh.t() / math.sqrt(D)
                prob = torch.softmax(x.masked_fill(hidden, float("-inf")), -1).masked_fill(empty, 0.0)
                o[b, h, a:a + len(p)] = prob @ vh
                if c["train"]:
                    g = s["do"][b, h, a:a + len(p)].double()
                    dv[b, h // G].index_add_(0, j, prob.t() @ g)
                    t = prob * (g @ vh.t())
                    t = (t - prob * t.sum(-1, keepdim=True)) / math.sqrt(D)
                    dq[b, h, a:a + len(p)] = t @ kh
                    dk[b, h // G].index_add_(0, j, t.t() @ qh)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if c["train"] else {"o": o}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "window": _exact_window}[case["op"]](case, s)
