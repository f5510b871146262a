"""Attention of packed sequences, MI355X implementation (csrc/packed_*.hip): the
sequences of a batch, of different lengths, stand behind one another in one tensor,
and each token sees its own sequence: prompts of a server, documents of a training
step.

Beside flash_attn_window, whose batches are padded to their longest sequence.  The
reference calls a dense attention library there (hymm/models/modules/
wan_video_dit.py:36-110).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops


def flash_attn_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
                      cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = True, sm_scale: Optional[float] = None,
                      return_lse: bool = False):
    """softmax(sm_scale q k^T) v within each sequence.

    q: [Tq, Hq, D], k, v: [Tk, Hk, D], bfloat16 or float16, D 64 or 128; Hq a multiple
    of Hk (query heads h * Hq / Hk .. share key head h).  Any strides; adjacent channels,
    16-byte aligned rows and strides of whole 16 bytes are read in place (parts of a
    projection's output), others are copied first.

    cu_seqlens: int32 [B + 1] on the GPU, not decreasing: sequence b's queries are rows
    cu_seqlens[b] to cu_seqlens[b + 1] - 1 of q, its keys the same rows of k and v, or
    those that cu_seqlens_k [B + 1] says (the next part of a prompt over all of its keys).
    Sequences may be empty; values outside the tensors are cut to them (where they
    decrease, nothing outside is read or written, but the results are not defined).  The
    queries are the last of their sequence: with L keys and n queries, query i sees keys j <= i + L - n
    (causal), or all.  Queries that see no key, and rows of no sequence, give 0, and take
    and give no gradient.  sm_scale (positive) defaults to D^-1/2.  A NaN or an infinity in
    a key or value reaches the queries that see it and no others (at about 1 us a key); in
    a backward pass it may reach the gradients of rows in the same tile of 64.

    Returns o, of q's shape (and layout, where q is dense), with return_lse (o, lse): lse
    [Hq, Tq] float32, the natural log of the sum of exponentials of the scaled scores, -inf
    where nothing is seen (no gradient through it).  Differentiable in q, k, v; sums over
    shared heads are fp32.  The backward keeps q, k, v, o, lse and what o's rounding left
    off, of o's size.  float16: P (dP - delta) beyond 1,023 becomes infinite, which a loss
    scaler sees.  No second and no forward-mode derivatives (refused)."""
    qs, ks, dt = q.shape, k.shape, q.dtype
    if len(qs) != 3 or len(ks) != 3 or ks != v.shape or ks[2] != qs[2]:
        raise ValueError(f"q must be [Tq, Hq, D], k and v [Tk, Hk, D], got {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}")
    Hq, D, Hk = qs[1], qs[2], ks[1]
    if D not in (64, 128):
        raise ValueError(f"head_dim {D} unsupported by the MI355X kernels (64, 128)")
    if Hk < 1 or Hq < Hk or Hq % Hk:
        raise ValueError(f"{Hq} query heads do not share {Hk} key heads evenly")
    if (dt is not torch.bfloat16 and dt is not torch.float16) or k.dtype is not dt or v.dtype is not dt:
        raise TypeError(f"q, k, v must be all bfloat16 or all float16, got {dt}, {k.dtype}, {v.dtype}")
    if cu_seqlens_k is None:
        if ks[0] != qs[0]:
            raise ValueError(f"{qs[0]} queries and {ks[0]} keys: keys of their own rows need cu_seqlens_k")
        cu_seqlens_k = cu_seqlens
    for t, name in ((cu_seqlens, "cu_seqlens"), (cu_seqlens_k, "cu_seqlens_k")):
        if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] < 1 or t.shape != cu_seqlens.shape:
            raise ValueError(f"{name} must be int32 [B + 1], got {t.dtype} {tuple(t.shape)}")
    sm_scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    if not 0 < sm_scale < float("inf"):
        raise ValueError(f"sm_scale must be positive and finite, got {sm_scale}")
    o, lse = ops.packed_fwd(q, k, v, cu_seqlens, cu_seqlens_k, causal, sm_scale, return_lse)
    return (o, lse) if return_lse else o


__all__ = ["flash_attn_packed"]
