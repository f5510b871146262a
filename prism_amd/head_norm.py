"""Root-mean-square norm of every query and key head, with its rotary positions in
the same pass, MI355X implementation (csrc/headnorm.hip):

    y = R(position) (x / sqrt(mean(x^2) + eps) * weight)

over the channels of a head: what a layer with head norms runs on its q and k
projections before the attention (the reference norms whole tokens,
hymm/models/modules/wan_video_dit.py:699-705; see rms_norm for that).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import ops


def qk_norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor], q_weight: Optional[torch.Tensor],
                   k_weight: Optional[torch.Tensor], freqs: torch.Tensor, positions: torch.Tensor, *, eps: float = 1e-6,
                   interleaved: bool = True, sections: Optional[Sequence[int]] = None, amplitude: float = 1.0):
    """q [B, Hq, S, D] and k [B, Hk, S, D] (or None), each head divided by the root
    of its mean square (plus eps), times its weight, then turned as apply_rotary
    does, in new tensors of the same layout.  float32, bfloat16 or float16, D up to
    256, at most 1,024 heads, any strides (best: adjacent channels).  q_weight,
    k_weight: [D] of q's dtype or float32 (both the same), or None for ones.  freqs,
    positions, interleaved, sections, amplitude: as for apply_rotary.  Returns q',
    with k (q', k').  Sums are fp32; results are rounded once (apply_rotary of a norm
    in between rounds twice).  A NaN makes all its head's results NaN; beside an infinity
    the root's inverse is 0, so that its own channel and the one that turns with it are
    NaN and the head's others 0; a sum of squares beyond float32 (values of 1.8e19 and
    more) makes a head 0.  No other head's results change (the weights' gradients are
    sums over all heads).  Differentiable in q, k and the weights (once; no forward
    mode; freqs that require gradients are refused)."""
    qs, ks, pairs = q.shape, None if k is None else k.shape, freqs.shape
    for s, name in ((qs, "q"), (ks, "k")):
        if s is not None and len(s) != 4:
            raise ValueError(f"qk_norm_rotary: {name} must be [B, H, S, D], got {tuple(s)}")
    if ks is not None and (ks[0] != qs[0] or ks[2:] != qs[2:]):
        raise ValueError(f"qk_norm_rotary: k {tuple(ks)} must have q's batch, length and head dim {tuple(qs)}")
    if not eps >= 0:
        raise ValueError(f"qk_norm_rotary: eps must not be negative, got {eps}")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is None:
            continue
        if w.shape != qs[3:]:
            raise ValueError(f"qk_norm_rotary: {name} must be [{qs[3]}], got {tuple(w.shape)}")
        if w.dtype not in (q.dtype, torch.float32):
            raise TypeError(f"qk_norm_rotary: {name} must have q's dtype {q.dtype} or float32, got {w.dtype}")
    if k is None and k_weight is not None:
        raise ValueError("qk_norm_rotary: k_weight without k")
    if q_weight is not None and k_weight is not None and q_weight.dtype is not k_weight.dtype:
        raise TypeError(f"qk_norm_rotary: q_weight and k_weight must have one dtype, got {q_weight.dtype} and {k_weight.dtype}")
    if freqs.dtype is not torch.float64:
        raise TypeError(f"qk_norm_rotary: freqs must be float64 (far positions lose their place in less), got {freqs.dtype}")
    if freqs.requires_grad and torch.is_grad_enabled():
        raise ValueError("qk_norm_rotary has no gradient for freqs: pass them detached")
    if len(pairs) != 1 or pairs[0] < 1 or 2 * pairs[0] > qs[3]:
        raise ValueError(f"qk_norm_rotary: {tuple(pairs)} frequencies do not fit heads of {qs[3]} channels")
    axis_pairs = []
    if sections is not None:
        if any(int(n) < 2 or int(n) % 2 for n in sections) or sum(int(n) for n in sections) != 2 * pairs[0]:
            raise ValueError(f"qk_norm_rotary: sections {list(sections)} must be even and sum to {2 * pairs[0]}")
        axis_pairs = [int(n) // 2 for n in sections]
    oq, ok = ops.qk_norm_rotary(q, k, q_weight, k_weight, eps, freqs, positions, axis_pairs, interleaved, amplitude)
    return oq if k is None else (oq, ok)


__all__ = ["qk_norm_rotary"]
