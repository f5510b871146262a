"""Attention over a sliding window and the first tokens (sinks), MI355X
implementation (csrc/window_*.hip): prompts and training steps, and single
tokens of a stream over its cache.

Beside the block-sparse attention, whose kept blocks follow the content, this
one's follow the position: the form for token streams (an audio tower, frames
generated one after the other), where each token sees the last `window` tokens
and the stream's first `sinks`.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops

_NO_LIMIT = 1 << 29  # a window that no sequence reaches


def flash_attn_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int], *, sinks: int = 0,
                      causal: bool = True, sm_scale: Optional[float] = None, q_lens: Optional[torch.Tensor] = None,
                      kv_lens: Optional[torch.Tensor] = None, return_lse: bool = False):
    """softmax(sm_scale q k^T) v over the keys that each query sees.

    q: [B, Hq, Sq, D], k, v: [B, Hk, Sk, D], bfloat16 or float16, D 64 or 128;
    Hq a multiple of Hk (query heads h * Hq / Hk .. share key head h).  Any
    strides; adjacent channels, 16-byte aligned rows and strides of whole 16
    bytes are read in place (a cache or a projection laid out [B, S, H, D],
    transposed), others are copied first.

    The queries are the last of their sequence: with L keys and n queries,
    query i stands at position p = i + L - n.  It sees key j < L where
      causal:      p - window < j <= p, or j < sinks and j <= p
      otherwise:   |p - j| < window, or j < sinks
    window None: no limit.  kv_lens, q_lens: int32 [B] on the GPU, L and n per
    sequence (default Sk and Sq; cut to them): a cache with room beyond its
    tokens, a batch padded on the right (both the same lengths).  Keys beyond L,
    and others that no query of the call sees, are not read and may hold
    anything.  Queries that see no key, and rows i >= n, give 0 (and take no
    gradient).  sm_scale (positive)
    defaults to D^-1/2.  A NaN or an infinity in a key or value reaches the
    queries that see it and no others (at about 1 us a key); in a backward pass
    it may reach the gradients of rows in the same tile of 64.

    Returns o, of q's shape (and layout, where q is dense), with return_lse (o,
    lse): lse [B, Hq, Sq] float32, the natural log of the sum of exponentials
    of the scaled scores, -inf where nothing is seen (no gradient through it).
    Differentiable in q, k, v; sums over shared heads are fp32.  The backward
    keeps q, k, v, o, lse and (where queries see more than 64 keys) what o's
    rounding left off, of o's size.  float16: P (dP - delta) beyond 1,023 becomes
    infinite, which a loss scaler sees.  No second and no forward-mode derivatives
    (refused)."""
    qs, ks, vs, dt = q.shape, k.shape, v.shape, q.dtype
    if len(qs) != 4 or len(ks) != 4 or len(vs) != 4:
        raise ValueError("q, k, v must be [B, H, S, D]")
    B, Hq, _, D = qs
    Hk = ks[1]
    if ks != vs or ks[0] != B or ks[3] != D:
        raise ValueError(f"shape mismatch: q {tuple(qs)}, k {tuple(ks)}, v {tuple(vs)}")
    if D not in (64, 128):
        raise ValueError(f"head_dim {D} unsupported by the MI355X kernels (64, 128)")
    if Hk < 1 or Hq < Hk or Hq % Hk:
        raise ValueError(f"{Hq} query heads do not share {Hk} key heads evenly")
    if (dt is not torch.bfloat16 and dt is not torch.float16) or k.dtype is not dt or v.dtype is not dt:
        raise TypeError(f"q, k, v must be all bfloat16 or all float16, got {dt}, {k.dtype}, {v.dtype}")
    if window is not None and int(window) < 1:
        raise ValueError(f"window must be at least 1 (or None), got {window}")
    if int(sinks) < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    for t, name in ((q_lens, "q_lens"), (kv_lens, "kv_lens")):
        if t is not None and (t.dtype is not torch.int32 or t.shape != (B,)):
            raise ValueError(f"{name} must be int32 [{B}], got {t.dtype} {tuple(t.shape)}")
    window = _NO_LIMIT if window is None else min(int(window), _NO_LIMIT)
    sinks = min(int(sinks), _NO_LIMIT)
    sm_scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    if not 0 < sm_scale < float("inf"):
        raise ValueError(f"sm_scale must be positive and finite, got {sm_scale}")
    o, lse = ops.window_fwd(q, k, v, window, sinks, causal, q_lens, kv_lens, sm_scale, return_lse)
    return (o, lse) if return_lse else o


__all__ = ["flash_attn_window"]
