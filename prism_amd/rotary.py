"""Rotary positions on queries and keys, MI355X implementation
(csrc/rotary.hip): what the model applies to q and k before the attention
(hymm/models/modules/wan_video_dit.py:699-705), there with the pairs of a head
shared out over the three axes of the video grid.

Pair p of a head's first 2 * len(freqs) channels is turned by position x
freqs[p] radians; channels past them are copied.  Frequencies are float64 and
angles are formed in float64, so far positions keep their place.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import ops


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, sections: Optional[Sequence[int]] = None,
                       scaling: Optional[str] = None, factor: float = 1.0, original_length: Optional[int] = None,
                       beta_fast: float = 32.0, beta_slow: float = 1.0, device="cuda"):
    """(freqs, amplitude) of apply_rotary for `rotary_dim` channels of a head:
    freqs [rotary_dim / 2] float64 on `device`, base^(-2i / rotary_dim) for pair
    i.  sections: even channel counts per axis (summing to rotary_dim), each
    axis with frequencies base^(-2i / its channels).  scaling, for contexts
    `factor` times longer than trained:
      "linear"  positions divided by factor;
      "ntk"     base grown by factor^(d / (d - 2)), so the slowest pair is
                divided by factor and the fastest is kept;
      "yarn"    pairs that turn beta_fast times or more within original_length
                kept, those that turn beta_slow times or less divided by
                factor, a linear ramp over the pair index between; amplitude
                0.1 ln(factor) + 1 (1 otherwise)."""
    parts = [int(n) for n in (sections if sections is not None else [rotary_dim])]
    if rotary_dim < 2 or rotary_dim % 2 or any(n < 2 or n % 2 for n in parts) or sum(parts) != rotary_dim:
        raise ValueError(f"rotary_dim {rotary_dim} and sections {parts} must be even, at least 2, and agree")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown rotary scaling: {scaling!r}")
    if not base > 1 or not factor >= 1:
        raise ValueError(f"base must be above 1 and factor at least 1, got {base} and {factor}")
    if scaling == "yarn" and (original_length is None or original_length < 1):
        raise ValueError("yarn scaling needs the original_length that the model was trained on")
    if scaling == "yarn" and not math.inf > beta_fast >= beta_slow > 0:
        raise ValueError(f"beta_fast must not be below beta_slow, and both positive, got {beta_fast} and {beta_slow}")
    amplitude, out = 1.0, []
    for d in parts:
        b = float(base)
        if scaling == "ntk":
            if d < 4:
                raise ValueError("ntk scaling needs sections of at least 4 channels")
            b *= factor ** (d / (d - 2.0))
        f = b ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        if scaling == "linear":
            f = f / factor
        elif scaling == "yarn":
            # pair index at which a pair turns n times within the original length
            def turns_at(n):
                return d * math.log(original_length / (n * 2 * math.pi)) / (2 * math.log(b))
            low = max(math.floor(turns_at(beta_fast)), 0)
            high = min(math.ceil(turns_at(beta_slow)), d - 1)  # (past the last pair where that turns more often)
            ramp = ((torch.arange(d // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
            f = f * (1 - ramp) + f / factor * ramp
            amplitude = 0.1 * math.log(factor) + 1.0
        out.append(f)
    return torch.cat(out).to(device), amplitude


def grid_positions(grid_size, device="cuda") -> torch.Tensor:
    """[T*H*W, 3] int32 (t, h, w) of the tokens of a T x H x W grid in THW order."""
    T, H, W = (int(n) for n in grid_size)
    at = torch.meshgrid(*[torch.arange(n, dtype=torch.int32, device=device) for n in (T, H, W)], indexing="ij")
    return torch.stack(at, dim=-1).view(T * H * W, 3)


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], freqs: torch.Tensor, positions: torch.Tensor, *,
                 interleaved: bool = True, sections: Optional[Sequence[int]] = None, amplitude: float = 1.0):
    """q [B, Hq, S, D] and k [B, Hk, S, D] (or None) turned by their tokens'
    positions, in new tensors of the same layout.  float32, bfloat16 or
    float16, D up to 256, any strides (best: adjacent channels).  freqs: float64
    [pairs] (rotary_frequencies), 2 * pairs <= D.  positions: int32 or int64
    [S] or [B, S]; with sections (channels per axis, summing to 2 * pairs, at
    most 4 axes) one entry per axis in a last dimension.  interleaved: pairs of
    channels (2p, 2p + 1), else (p, p + pairs).  amplitude scales the turned
    channels.  Returns q', with k (q', k').  Differentiable in q and k (once; no
    forward mode; freqs that require gradients are refused)."""
    qs, ks, pairs = q.shape, None if k is None else k.shape, freqs.shape
    for s, name in ((qs, "q"), (ks, "k")):
        if s is not None and len(s) != 4:
            raise ValueError(f"apply_rotary: {name} must be [B, H, S, D], got {tuple(s)}")
    if ks is not None and (ks[0] != qs[0] or ks[2:] != qs[2:]):
        raise ValueError(f"apply_rotary: k {tuple(ks)} must have q's batch, length and head dim {tuple(qs)}")
    if freqs.dtype is not torch.float64:
        raise TypeError(f"apply_rotary: freqs must be float64 (far positions lose their place in less), got {freqs.dtype}")
    if freqs.requires_grad and torch.is_grad_enabled():
        raise ValueError("apply_rotary has no gradient for freqs: pass them detached")
    if len(pairs) != 1 or pairs[0] < 1 or 2 * pairs[0] > qs[3]:
        raise ValueError(f"apply_rotary: {tuple(pairs)} frequencies do not fit heads of {qs[3]} channels")
    axis_pairs = []
    if sections is not None:
        if any(int(n) < 2 or int(n) % 2 for n in sections) or sum(int(n) for n in sections) != 2 * pairs[0]:
            raise ValueError(f"apply_rotary: sections {list(sections)} must be even and sum to {2 * pairs[0]}")
        axis_pairs = [int(n) // 2 for n in sections]
    oq, ok = ops.rotary(q, k, freqs, positions, axis_pairs, interleaved, amplitude)
    return oq if k is None else (oq, ok)


__all__ = ["rotary_frequencies", "grid_positions", "apply_rotary"]
