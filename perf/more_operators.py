"""Timed cases of the operators of packed batches and paged caches: what a layer
runs when its sequences stand behind one another in one tensor, and when their
keys and values stand in pages that the sequences share.

  qknorm   qk_norm_rotary: root-mean-square norm of every query and key head and
           its rotary positions
  packed   flash_attn_packed: attention of packed sequences of different lengths,
           shared key heads, causal; prompts and training steps
  append   append_paged (and gather_paged, which reads sequences back): keys,
           turned by their positions, and values into a paged cache of 16-bit
           elements or of 4-bit elements with a scale for each 32
  paged    flash_attn_paged: new tokens over such a cache

``listed`` holds the named cases, ``draw`` makes others of the same ranges,
``prepare`` makes a case's inputs, ``run`` makes one pass (where ``own`` is
false in plain torch operations, rounded once at the end; where it is true
through the framework's entry points), ``work`` counts what a pass cannot do
without and ``exact`` computes it in 64 bits.

A paged cache is two tensors (keys, values).  16 bits: [pages, heads, page size,
D].  4 bits: uint8 [pages, heads, page size (D / 2 + D / 32)]: the codes of a
page's places, D / 2 bytes each (an even channel in the low half of its byte),
then their scales, D / 32 bytes each.  A code is a sign and one of 0, 0.5, 1, 1.5,
2, 3, 4, 6; a scale byte e stands for 2^(e - 127), the least that keeps 32 channels
within 6 (1 at least; 255 where one is not finite).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases
def _qknorm(B, S, Hq, Hk, D, *, rotary_dim=None, interleaved=True, axes="", scaling="none", far=0, dtype="bf16",
            projected=False, train=False, name=None):
    """axes: "" for one position a token, else "TxHxW" (S tokens of that grid);
    far: the first position; projected: [B, S, H, D] in memory."""
    c = dict(op="qknorm", B=B, S=S, Hq=Hq, Hk=Hk, D=D, rotary_dim=rotary_dim or D, interleaved=interleaved, axes=axes,
             scaling=scaling, far=far, dtype=dtype, projected=projected, train=train)
    return dict(c, name=name) if name else c


def _packed(B, T, Hq, Hk, D, *, causal=True, dtype="bf16", train=False, name=None):
    """T tokens of B sequences, each half to one and a half times their mean."""
    c = dict(op="packed", B=B, T=T, Hq=Hq, Hk=Hk, D=D, causal=causal, dtype=dtype, train=train)
    return dict(c, name=name) if name else c


def _append(B, T, room, Hk, D, page, *, bits=16, read=False, interleaved=False, dtype="bf16", name=None):
    """T new tokens of B sequences (each one's share as in packed; T = B: one
    each) behind 3/4 `room` that are there in the mean; read: the sequences are read back."""
    c = dict(op="append", B=B, T=T, room=room, Hk=Hk, D=D, page=page, bits=bits, read=read, interleaved=interleaved,
             dtype=dtype)
    return dict(c, name=name) if name else c


def _paged(B, n, L, Hq, Hk, D, page, *, bits=16, dtype="bf16", name=None):
    """n new tokens of each of B sequences of L / 2 to L tokens."""
    c = dict(op="paged", B=B, n=n, L=L, Hq=Hq, Hk=Hk, D=D, page=page, bits=bits, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One new token of each of 16 streams, far beyond the trained length:
        # latency.
        _qknorm(16, 1, 32, 8, 128, interleaved=False, scaling="yarn", far=200000, name="qknorm_token"),
        # Queries and keys of a 720p clip (21 x 45 x 80 latent tokens), 40 heads,
        # as the projections leave them, three axes, inference: bandwidth.
        _qknorm(1, 75600, 40, 40, 128, axes="21x45x80", projected=True, name="qknorm_720p"),
        # A training step of a text batch: part of a small head, an odd length.
        _qknorm(2, 4999, 16, 4, 64, rotary_dim=32, interleaved=False, scaling="linear", projected=True, train=True,
                name="qknorm_part_train"),
        # A few short questions that a server has gathered: latency.
        _packed(7, 301, 32, 8, 128, name="packed_short"),
        # Prompts of a busy server, an odd total.
        _packed(3, 16001, 32, 8, 128, name="packed_prompts"),
        # A training step over packed documents.
        _packed(6, 8191, 16, 4, 128, train=True, name="packed_train"),
        # One new token of each of 32 streams into pages of 16: latency.
        _append(32, 32, 4096, 8, 128, 16, name="append_token"),
        # New prompts into 16-bit pages.
        _append(3, 16001, 0, 8, 128, 64, interleaved=True, name="append_prompts"),
        # The next part of long prompts into 4-bit pages, and the sequences read
        # back for its attention.
        _append(4, 8191, 8192, 8, 128, 32, bits=4, read=True, name="append_part_4bit"),
        # One new token of each of 16 streams of different lengths.
        _paged(16, 1, 8192, 32, 8, 128, 16, name="paged_token"),
        # Three proposed tokens of a few streams, small heads, 4-bit pages:
        # latency.
        _paged(4, 3, 2000, 16, 4, 64, 32, bits=4, dtype="fp16", name="paged_proposed_4bit"),
        # Long streams over 4-bit pages: bandwidth.
        _paged(8, 1, 131072, 32, 8, 128, 64, bits=4, name="paged_long_4bit"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qknorm", "packed", "packed", "append", "paged", "paged"])
    train = rng.random() < 0.45
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    Hk = rng.choice([1, 2, 4, 5, 8])
    Hq = Hk * rng.choice([1, 1, 2, 3, 4, 8])
    B = rng.choice([1, 1, 2, 3, 5, 8, 17, 70])
    if op == "qknorm":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        D = rng.choice([32, 64, 64, 80, 128, 128, 128, 256])
        part = rng.choice([D, D, D, D // 2, D // 4])
        B, axes = min(B, 8), ""
        S = _log(rng, 1, min(40000, 2.5e8 / (B * Hq * D)))
        if rng.random() < 0.35:
            T, H, W = rng.randint(1, 13), rng.randint(3, 45), rng.randint(4, 60)
            axes, S, part, B = "%dx%dx%d" % (T, H, W), T * H * W, D, 1
        return _qknorm(B, S, Hq, Hk, D, rotary_dim=part, interleaved=rng.random() < 0.5, axes=axes,
                       scaling="none" if axes else rng.choice(["none", "linear", "ntk", "yarn"]),
                       far=0 if axes else rng.choice([0, 0, 777, 300000]), dtype=dtype,
                       projected=rng.random() < 0.5, train=train)
    D = rng.choice([64, 128, 128])
    if op == "packed":
        T = _log(rng, B, max(64 * B, min(16001, math.sqrt(6e8 * B / Hq))))
        return _packed(B, T, Hq, Hk, D, causal=rng.random() < 0.75, dtype=dtype, train=train)
    page, bits = rng.choice([16, 16, 32, 64, 128, 256]), rng.choice([16, 16, 4])
    if op == "append":
        T = B if rng.random() < 0.4 else _log(rng, B, max(2 * B, 16001))
        room = rng.choice([0, 0, _log(rng, 1, max(2, 60000 // B))])
        return _append(B, T, room, Hk, D, page, bits=bits, read=bits == 4 or rng.random() < 0.4,
                       interleaved=rng.random() < 0.5, dtype=dtype)
    return _paged(B, rng.choice([1, 1, 1, 2, 5]), _log(rng, 1, 500000 // B), Hq, Hk, D, page, bits=bits, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _frequencies(c):
    """float64 angle per position of every pair, and the factor on the rotated
    channels (scalings: 8 times a trained length of 8,192)."""
    R, base, factor, trained = c.get("rotary_dim", c["D"]), 10000.0, 8.0, 8192
    if c.get("axes"):
        return torch.cat([base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n) for n in _sections(R)]), 1.0
    i, scaling = torch.arange(0, R, 2, dtype=torch.float64), c.get("scaling")
    if scaling == "ntk":
        return (base * factor ** (R / (R - 2.0))) ** (-i / R), 1.0
    f = base ** (-i / R)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":  # pairs that turn 32 times or more in the trained length stay, below once are divided
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


def _shares(seed, B, T):
    """Lengths of B sequences of T tokens in all, half to one and a half times
    their mean (one or none where there are few)."""
    rng = random.Random(seed)
    w = [rng.uniform(0.5, 1.5) for _ in range(B)]
    at = [int(round(T * sum(w[:i]) / sum(w))) for i in range(B)] + [T]
    return [b - a for a, b in zip(at, at[1:])]


def _starts(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def _device(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _pages(seed, lens, page):
    """A page table of sequences of these lengths over pages in any order (-1
    behind a sequence's last), and how many pages there are."""
    need = [-(-n // page) for n in lens]
    pages = sum(lens) // page + len(lens) + 3
    ids = list(range(pages))
    random.Random(seed).shuffle(ids)
    wide, table = max(max(need), 1), []
    for n in need:
        table.append(ids[:n] + [-1] * (wide - n))
        ids = ids[n:]
    return _device(table), pages


def _filled(g, pages, c):
    """A cache of these many pages that holds something."""
    dt, D, page, Hk = DTYPES[c["dtype"]], c["D"], c["page"], c["Hk"]
    if c["bits"] == 16:
        return [torch.randn(pages, Hk, page, D, generator=g, device=DEVICE, dtype=dt) for _ in "kv"]
    out = []
    for _ in "kv":
        parts = []
        for a in range(0, pages, 4096):
            x = torch.randn(min(4096, pages - a), Hk, page, D, generator=g, device=DEVICE)
            x[..., ::29] *= 3  # a few larger channels
            codes, scales = _to_4bit(x)
            parts.append(torch.cat([codes.flatten(2), scales.flatten(2)], -1))
        out.append(torch.cat(parts))
    return out


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rand = lambda *shape, dtype=DTYPES[c["dtype"]]: torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)  # noqa: E731
    s = {"case": c}
    B, Hk, D = c["B"], c["Hk"], c["D"]
    if c["op"] == "qknorm":
        S = c["S"]

        def heads(H):
            return rand(B, S, H, D).transpose(1, 2) if c["projected"] else rand(B, H, S, D)
        s["q"], s["k"] = heads(c["Hq"]), heads(Hk)
        s["k"][..., ::29] *= 4  # a few channels far larger
        s["wq"], s["wk"] = ((torch.rand(D, generator=g, device=DEVICE) + 0.5).to(s["q"].dtype) for _ in "qk")
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
            s["dq"], s["dk"] = heads(c["Hq"]), heads(Hk)
        return s
    if c["op"] == "packed":
        T, s["lens"] = c["T"], _shares(seed, B, c["T"])
        s["starts"] = _device(_starts(s["lens"]))
        s["q"], s["k"], s["v"] = rand(T, c["Hq"], D), rand(T, Hk, D), rand(T, Hk, D)
        if c["train"]:
            s["do"] = rand(T, c["Hq"], D)
        return s
    if c["op"] == "append":
        s["new"] = _shares(seed, B, c["T"]) if c["T"] != B else [1] * B
        s["lens"] = [n + m for n, m in zip(s["new"], _shares(seed + 1, B, 3 * B * c["room"] // 4))]
        s["starts"] = _device(_starts(s["new"])) if c["T"] != B else None
        s["read_starts"] = _device(_starts(s["lens"]))
        s["k"], s["v"] = rand(c["T"], Hk, D), rand(c["T"], Hk, D)
        s["k"][..., ::29] *= 3
        s["freqs"] = _frequencies(c)[0].to(DEVICE)
    else:
        rng = random.Random(seed + 1)
        s["lens"] = [rng.randint(max(1, c["L"] // 2), c["L"]) for _ in range(B)]
        s["q"] = rand(B * c["n"], c["Hq"], D)
    s["kv_lens"] = _device(s["lens"])
    s["table"], pages = _pages(seed + 2, s["lens"], c["page"])
    s["kc"], s["vc"] = _filled(g, pages, c)
    return s


# ------------------------------------------------------------------ one pass: norms and positions of heads
def _turn(c, x, cos, sin):
    """fp32 or fp64 [.., D] turned by the angles of cos, sin [.., R/2]."""
    R = c.get("rotary_dim", c["D"])
    rot, rest = x[..., :R], x[..., R:]
    if c["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = rot[..., :R // 2], rot[..., R // 2:]
        rot = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([rot, rest], -1)


def _plain_qknorm(c, s):
    p, dt, eps = s["positions"], DTYPES[c["dtype"]], 1e-6
    if c["axes"]:
        n = torch.tensor([m // 2 for m in _sections(c["rotary_dim"])])
        axis = torch.repeat_interleave(torch.arange(3), n).to(DEVICE)
        angle = p.double()[:, axis] * s["freqs"]  # [S, R/2]
    else:
        angle = (p.double()[..., None] * s["freqs"])[:, None]  # [B, 1, S, R/2]
    cos, sin = (t.mul(s["amplitude"]).float() for t in (angle.cos(), angle.sin()))

    def one(x, w, dy):
        x, w = x.float(), w.float()
        inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        xh = x * inv
        y = _turn(c, xh * w, cos, sin).to(dt)
        if not c["train"]:
            return y, None, None
        gy = _turn(c, dy.float(), cos, -sin)
        gx = gy * w
        return y, (inv * (gx - xh * (gx * xh).mean(-1, keepdim=True))).to(dt), (gy * xh).sum((0, 1, 2)).to(dt)

    q, dq, dwq = one(s["q"], s["wq"], s.get("dq"))
    k, dk, dwk = one(s["k"], s["wk"], s.get("dk"))
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk} if c["train"] else {"q": q, "k": k}


def _own_qknorm(c, s):
    import prism_amd
    kw = dict(eps=1e-6, interleaved=c["interleaved"], amplitude=s["amplitude"],
              sections=_sections(c["rotary_dim"]) if c["axes"] else None)
    if not c["train"]:
        q, k = prism_amd.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["freqs"], s["positions"], **kw)
        return {"q": q, "k": k}
    leaves = [s[n].detach().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
    q, k = prism_amd.qk_norm_rotary(*leaves, s["freqs"], s["positions"], **kw)
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), leaves, (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


# ------------------------------------------------------------------ one pass: packed attention
def _plain_packed(c, s):
    B, T, Hq, Hk, D = (c[n] for n in ("B", "T", "Hq", "Hk", "D"))
    dt, G, scale, N = DTYPES[c["dtype"]], Hq // Hk, 1.0 / math.sqrt(D), max(s["lens"])
    first, i = s["starts"].long(), torch.arange(N, device=DEVICE)
    n = first[1:] - first[:-1]
    there = i < n[:, None]  # [B, N]
    at = (first[:-1, None] + i).clamp(max=T - 1)

    def pad(t):  # [T, H, D] -> [B, Hk, G N, D], zeros behind a sequence's end
        x = t.float()[at].masked_fill_(~there[..., None, None], 0.0)
        return x.view(B, N, Hk, -1, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)

    def unpad(x, H):  # and back
        return x.view(B, Hk, H // Hk, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H, D)[there].to(dt)

    q, k, v = pad(s["q"]), pad(s["k"]), pad(s["v"])
    x = (q @ k.transpose(-1, -2).contiguous()).mul_(scale).view(B, Hk, G, N, N)
    seen = there[:, None, :]  # [B, N, N]
    if c["causal"]:
        seen = seen & (i[:, None] >= i)
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    e = x.sub_(top.masked_fill(torch.isinf(top), 0.0)).exp_()
    p = e.div_(e.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, Hk, G * N, N)
    o = p @ v
    out = {"o": unpad(o, Hq)}
    if c["train"]:
        do = pad(s["do"])
        dv = p.transpose(-1, -2).contiguous() @ do
        ds = (do @ v.transpose(-1, -2).contiguous()).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"], out["dv"] = unpad(ds @ k, Hq), unpad(dv, Hk)
        out["dk"] = unpad(ds.transpose(-1, -2).contiguous() @ q, Hk)
    return out


def _own_packed(c, s):
    import prism_amd
    if not c["train"]:
        return {"o": prism_amd.flash_attn_packed(s["q"], s["k"], s["v"], s["starts"], causal=c["causal"])}
    q, k, v = (s[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
    o = prism_amd.flash_attn_packed(q, k, v, s["starts"], causal=c["causal"])
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


# ------------------------------------------------------------------ one pass: the paged cache
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _to_4bit(x):
    """Codes [.., D/2] and scales [.., D/32] (uint8) of x [.., D]."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e, 0.5 <= m < 1; 6 = 0.75 2^3
    byte = (e + 124 + (m > 0.75).int()).clamp(1, 254)
    byte = torch.where(torch.isfinite(top), torch.where(top > 0, byte, torch.ones_like(byte)), torch.full_like(byte, 255))
    z = torch.ldexp(b, 127 - byte[..., None].float())
    a = z.abs().nan_to_num(0.0, 0.0)
    # (rint: halves to even, and every second level has an even code)
    level = torch.where(a < 2, (2 * a).round(), torch.where(a < 4, a.round() + 2, (a / 2).round() + 4))
    code = (level.clamp(max=7).to(torch.uint8) | (torch.signbit(z).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _of_4bit(codes, scales):
    """fp32 values of codes [.., D/2] and scales [.., D/32]."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=DEVICE)
    pair = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return torch.ldexp(levels[pair].unflatten(-1, (-1, 32)), scales[..., None].float() - 127).flatten(-2)


def _split_4bit(c, cache):
    """The codes [P, Hk, page, D/2] and scales [P, Hk, page, D/32] of a cache (views)."""
    P, Hk, page, D = cache.shape[0], c["Hk"], c["page"], c["D"]
    return (cache[..., :page * D // 2].view(P, Hk, page, D // 2), cache[..., page * D // 2:].view(P, Hk, page, D // 32))


def _rows(c, cache, where, place):
    """fp32 rows [.., Hk, D] of pages `where` at places `place`."""
    if c["bits"] == 16:
        return cache[where, :, place].float()
    codes, scales = _split_4bit(c, cache)
    return _of_4bit(codes[where, :, place], scales[where, :, place])


def _plain_append(c, s):
    B, T, page, dt = c["B"], c["T"], c["page"], DTYPES[c["dtype"]]
    first = s["starts"].long() if s["starts"] is not None else torch.arange(B + 1, device=DEVICE)
    n = first[1:] - first[:-1]
    who = torch.repeat_interleave(torch.arange(B, device=DEVICE), n, output_size=T)
    at = s["kv_lens"].long()[who] - n[who] + torch.arange(T, device=DEVICE) - first[who]  # places, and positions
    where, place = s["table"][who, at // page].long(), at % page
    angle = at.double()[:, None, None] * s["freqs"]
    if c["bits"] == 16:
        k = _turn(c, s["k"].float(), angle.cos().float(), angle.sin().float()).to(dt)
        s["kc"][where, :, place], s["vc"][where, :, place] = k, s["v"]
        out = {"k_cache": s["kc"], "v_cache": s["vc"]}
    else:  # (64 bits: a value beside a border between two codes is rounded to the right one)
        k = _turn(c, s["k"].double(), angle.cos(), angle.sin()).to(dt)
        for cache, x in ((s["kc"], k), (s["vc"], s["v"])):
            for part, new in zip(_split_4bit(c, cache), _to_4bit(x)):
                part[where, :, place] = new
        out = {}
    if c["read"]:
        total = sum(s["lens"])
        first = s["read_starts"].long()
        who = torch.repeat_interleave(torch.arange(B, device=DEVICE), s["kv_lens"].long(), output_size=total)
        at = torch.arange(total, device=DEVICE) - first[who]
        where, place = s["table"][who, at // page].long(), at % page
        out["k"], out["v"] = _rows(c, s["kc"], where, place).to(dt), _rows(c, s["vc"], where, place).to(dt)
    return out


def _own_append(c, s):
    import prism_amd
    prism_amd.append_paged(s["k"], s["v"], s["kc"], s["vc"], s["table"], s["kv_lens"], cu_seqlens=s["starts"],
                           freqs=s["freqs"], interleaved=c["interleaved"])
    out = {"k_cache": s["kc"], "v_cache": s["vc"]} if c["bits"] == 16 else {}
    if c["read"]:
        out["k"], out["v"] = prism_amd.gather_paged(s["kc"], s["vc"], s["table"], s["read_starts"], sum(s["lens"]),
                                                    head_dim=c["D"], dtype=s["k"].dtype)
    return out


def _plain_paged(c, s):
    B, n, Hq, Hk, D, page = (c[x] for x in ("B", "n", "Hq", "Hk", "D", "page"))
    G, N = Hq // Hk, max(s["lens"])
    at = torch.arange(N, device=DEVICE)
    where = s["table"].long().clamp(min=0)[:, at // page]  # [B, N]
    k, v = (_rows(c, s[x], where, (at % page).expand(B, N)).transpose(1, 2).contiguous() for x in ("kc", "vc"))
    q = s["q"].float().view(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * n, D)
    x = (q @ k.transpose(-1, -2).contiguous()).div_(math.sqrt(D)).view(B, Hk, G, n, N)
    last = s["kv_lens"].long()[:, None] - n + torch.arange(n, device=DEVICE)  # [B, n]
    x.masked_fill_((at > last[..., None])[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    e = x.sub_(top.masked_fill(torch.isinf(top), 0.0)).exp_()
    p = e.div_(e.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, Hk, G * n, N)
    o = (p @ v).view(B, Hk, G, n, D).permute(0, 3, 1, 2, 4).reshape(B * n, Hq, D)
    return {"o": o.to(s["q"].dtype)}


def _own_paged(c, s):
    import prism_amd
    return {"o": prism_amd.flash_attn_paged(s["q"], s["kc"], s["vc"], s["table"], s["kv_lens"])}


_PLAIN = {"qknorm": _plain_qknorm, "packed": _plain_packed, "append": _plain_append, "paged": _plain_paged}
_OWN = {"qknorm": _own_qknorm, "packed": _own_packed, "append": _own_append, "paged": _own_paged}


def run(state):
    c = state["case"]
    return (_OWN if own else _PLAIN)[c["op"]](c, state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Inputs read once and outputs written once.  qknorm: 9 operations an element
    forward, 17 more backward.  packed: 4 D operations a seen pair, 14 D with the
    backward, sequences at their mean.  append: the rotation's 3 operations a key
    element; what is read back is read and written.  paged: lengths at their mean."""
    c = case
    es, B, Hk, D = BYTES[c["dtype"]], c["B"], c["Hk"], c["D"]
    if c["op"] == "qknorm":
        n = float(B) * c["S"] * (c["Hq"] + Hk) * D
        b = 2 * es * n + 8.0 * B * c["S"]
        return {"bytes": b + 2 * es * n if c["train"] else b, "flops": (26 if c["train"] else 9) * n}
    if c["op"] == "packed":
        # (lengths w mean, w uniform on 0.5 .. 1.5: their squares' mean is 13 / 12)
        T, mean = float(c["T"]), c["T"] / B
        pairs = T * c["Hq"] * (mean * 13 / 12 if B > 1 else mean) * (0.5 if c["causal"] else 1.0)
        b = es * D * T * (2 * c["Hq"] + 2 * Hk)
        return {"bytes": 2 * b if c["train"] else b, "flops": max(1.0, pairs) * D * (14 if c["train"] else 4)}
    row = 2 * D if c["bits"] == 16 else D / 2 + D / 32
    if c["op"] == "append":
        T = float(c["T"])
        b = Hk * T * 2 * (es * D + row)
        if c["read"]:
            b += Hk * (T + 0.75 * c["room"] * B) * 2 * (row + es * D)
        return {"bytes": b, "flops": 3 * T * Hk * D}
    keys = max(1.0, 0.75 * c["L"])
    return {"bytes": B * (2 * Hk * keys * row + 2 * es * c["n"] * c["Hq"] * D),
            "flops": 4.0 * D * B * c["n"] * c["Hq"] * keys}


# ------------------------------------------------------------------ float64
def _exact_turn(c, x, unit):
    """x [.., D] (float64) times the complex numbers of unit [.., R/2], pair by pair."""
    R = c.get("rotary_dim", c["D"])
    y, z = x.clone(), x[..., :R]
    pair = z.unflatten(-1, (R // 2, 2)) if c["interleaved"] else z.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    z2 = torch.view_as_real(torch.complex(pair[..., 0].contiguous(), pair[..., 1].contiguous()) * unit)
    y[..., :R] = z2.flatten(-2) if c["interleaved"] else z2.transpose(-1, -2).flatten(-2)
    return y


def _exact_qknorm(c, s):
    one = torch.tensor(1.0, dtype=torch.float64, device=DEVICE)
    p = s["positions"].double()
    if c["axes"]:
        n = [m // 2 for m in _sections(c["rotary_dim"])]
        angle = torch.cat([p[:, a:a + 1] * f for a, f in enumerate(torch.split(s["freqs"], n))], -1)[None]
    else:
        angle = p[..., None] * s["freqs"]
    unit = torch.polar(one, angle) * s["amplitude"]  # [B or 1, S, R/2]
    out = {}
    for x, w, g in (("q", "wq", "dq"), ("k", "wk", "dk")):
        y, dx = (torch.empty(s[x].shape, dtype=torch.float64, device=DEVICE) if t else None for t in (True, c["train"]))
        dw = torch.zeros(c["D"], dtype=torch.float64, device=DEVICE)
        weight = s[w].double()
        for h in range(s[x].shape[1]):
            v = s[x][:, h].double()
            length = (v.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt()
            y[:, h] = _exact_turn(c, v / length * weight, unit)
            if c["train"]:
                back = _exact_turn(c, s[g][:, h].double(), unit.conj())
                dw += (back * v / length).sum((0, 1))
                back = back * weight
                dx[:, h] = back / length - v * (back * v).sum(-1, keepdim=True) / (c["D"] * length.pow(3))
        out[x] = y
        if c["train"]:
            out[g], out["d" + w] = dx, dw
    return out


def _exact_packed(c, s):
    """One sequence, one head and a run of queries at a time."""
    Hq, Hk, D, T = (c[n] for n in ("Hq", "Hk", "D", "T"))
    G, run_of = Hq // Hk, 2048
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=DEVICE)
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(T, Hk, D, dtype=torch.float64, device=DEVICE) for _ in "kv")
    first = 0
    for n in s["lens"]:
        end = first + n
        for a in range(first, end, run_of):
            b = min(a + run_of, end)
            upto = b if c["causal"] else end
            hidden = None
            if c["causal"]:
                hidden = torch.arange(first, upto, device=DEVICE)[None] > torch.arange(a, b, device=DEVICE)[:, None]
            for h in range(Hq):
                qh, kh, vh = s["q"][a:b, h].double(), s["k"][first:upto, h // G].double(), s["v"][first:upto, h // G].double()
                x = qh @ kh.t() / math.sqrt(D)
                prob = torch.softmax(x if hidden is None else x.masked_fill(hidden, float("-inf")), -1)
                o[a:b, h] = prob @ vh
                if c["train"]:
                    g = s["do"][a:b, h].double()
                    dv[first:upto, h // G] += prob.t() @ g
                    t = prob * (g @ vh.t())
                    t = (t - prob * t.sum(-1, keepdim=True)) / math.sqrt(D)
                    dq[a:b, h] = t @ kh
                    dk[first:upto, h // G] += t.t() @ qh
        first = end
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if c["train"] else {"o": o}


def _exact_levels(x):
    """What 4 bits hold of x [.., D], by its definition: the nearest of scale x
    level, the even code where two are as near."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -300)
    scale = torch.exp2(torch.ceil(torch.log2(top / 6.0)))
    scale = torch.where(top > 6 * scale, 2 * scale, torch.where(top <= 3 * scale, scale / 2, scale))  # (log2's own rounding)
    scale = scale.clamp(min=2.0 ** -126)
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=DEVICE)
    z = b.abs() / scale
    low = (torch.searchsorted(levels, z.contiguous(), right=True) - 1).clamp(0, 6)
    under, over = z - levels[low], levels[low + 1] - z
    up = (over < under) | ((over == under) & (low % 2 == 1))
    return (levels[low + up.long()] * scale * torch.where(b < 0, -1.0, 1.0)).flatten(-2)


def _exact_place(c, s, cache, b, at):
    """float64 rows [len(at), Hk, D] of sequence b."""
    D, page = c["D"], c["page"]
    where, place = s["table"][b].long()[torch.div(at, page, rounding_mode="floor")], at % page
    if c["bits"] == 16:
        return cache[where, :, place].double()
    code = cache[where][..., :page * D // 2].view(len(at), c["Hk"], page, D // 2)
    byte = cache[where][..., page * D // 2:].view(len(at), c["Hk"], page, D // 32)
    i = torch.arange(len(at), device=DEVICE)
    code, byte = code[i, :, place].long(), byte[i, :, place].double()
    y = torch.empty(*code.shape[:-1], D, dtype=torch.float64, device=DEVICE)
    for half in (0, 1):
        nibble = (code >> (4 * half)) & 15
        size = torch.tensor(LEVELS, dtype=torch.float64, device=DEVICE)[nibble & 7]
        y[..., half::2] = torch.where(nibble > 7, -size, size)
    return y * torch.exp2(byte - 127).repeat_interleave(32, -1)


def _exact_append(c, s):
    dt, out = DTYPES[c["dtype"]], {}
    one = torch.tensor(1.0, dtype=torch.float64, device=DEVICE)
    new, old = {"k": [], "v": []}, {"k": [], "v": []}
    caches = {"k": s["kc"].double(), "v": s["vc"].double()} if c["bits"] == 16 else {}
    first = 0
    for b, (n, L) in enumerate(zip(s["new"], s["lens"])):
        at = torch.arange(L - n, L, device=DEVICE)
        unit = torch.polar(one, at.double()[:, None] * s["freqs"])[:, None]
        k = _exact_turn(c, s["k"][first:first + n].double(), unit)
        v = s["v"][first:first + n].double()
        for x, rows in (("k", k), ("v", v)):
            for a in range(0, L - n, 4096) if c["read"] else ():
                old[x].append(_exact_place(c, s, s[x + "c"], b, torch.arange(a, min(a + 4096, L - n), device=DEVICE)))
            old[x].append(rows if c["bits"] == 16 else _exact_levels(rows.to(dt)))
            if caches:
                where = s["table"][b].long()[torch.div(at, c["page"], rounding_mode="floor")]
                caches[x][where, :, at % c["page"]] = rows
        first += n
    if caches:
        out["k_cache"], out["v_cache"] = caches["k"], caches["v"]
    if c["read"]:
        out["k"], out["v"] = torch.cat(old["k"]), torch.cat(old["v"])
    return out


def _exact_paged(c, s):
    """One sequence after the other, its keys in parts with a running sum."""
    B, n, Hq, Hk, D = (c[x] for x in ("B", "n", "Hq", "Hk", "D"))
    G, part = Hq // Hk, 4096
    o = torch.zeros(B * n, Hq, D, dtype=torch.float64, device=DEVICE)
    for b, L in enumerate(s["lens"]):
        q = s["q"][b * n:b * n + n].double().view(n, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * n, D)
        last = (L - n + torch.arange(n, device=DEVICE)).repeat(G)[:, None]
        m = torch.full((Hk, G * n, 1), -1e300, dtype=torch.float64, device=DEVICE)
        total, acc = torch.zeros_like(m), torch.zeros_like(q)
        for a in range(0, L, part):
            at = torch.arange(a, min(a + part, L), device=DEVICE)
            k, v = (_exact_place(c, s, s[x], b, at).permute(1, 0, 2).contiguous() for x in ("kc", "vc"))
            x = (q @ k.transpose(1, 2).contiguous() / math.sqrt(D)).masked_fill(at > last, float("-inf"))
            top = torch.maximum(m, x.amax(-1, keepdim=True))
            e, f = torch.exp(x - top), torch.exp(m - top)
            m, total, acc = top, total * f + e.sum(-1, keepdim=True), acc * f + e @ v
        seen = total > 0
        o[b * n:b * n + n] = torch.where(seen, acc / torch.where(seen, total, 1.0), 0.0).view(Hk, G, n, D).permute(
            2, 0, 1, 3).reshape(n, Hq, D)
    return {"o": o}


def exact(case, seed):
    s = prepare(case, seed)
    return {"qknorm": _exact_qknorm, "packed": _exact_packed, "append": _exact_append,
            "paged": _exact_paged}[case["op"]](case, s)
