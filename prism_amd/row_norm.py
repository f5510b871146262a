"""Root-mean-square norm of token rows with the residual's addition, MI355X
implementation (csrc/rownorm.hip).

The model norms what enters its projections (hymm/models/modules/
wan_video_dit.py:699-705 norms q and k before the attention):

    h = x + residual,   y = h / sqrt(mean(h^2) + eps) * weight

One pass over the rows gives h (the residual stream that goes on), y, and where
the next product takes 8 bits, y's codes with one scale per row.  Sums are
fp32; y is formed from the unrounded sum and rounded once.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops


def _check(x, weight, residual, eps, name):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: x must have a last dimension of at least 1, got {tuple(x.shape)}")
    if not eps >= 0:
        raise ValueError(f"{name}: eps must not be negative, got {eps}")
    if weight is not None:
        if weight.shape != x.shape[-1:]:
            raise ValueError(f"{name}: weight must be [{x.shape[-1]}], got {tuple(weight.shape)}")
        if weight.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name}: weight must have x's dtype {x.dtype} or float32, got {weight.dtype}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{name}: residual {tuple(residual.shape)} must have x's shape {tuple(x.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError(f"{name}: residual must have x's dtype {x.dtype}, got {residual.dtype}")


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension, h = x +
    residual.  x: [..., N] (N up to 16,384) float32, bfloat16 or float16;
    weight: [N] of x's dtype or float32, or None for ones; residual: x's shape
    and dtype, or None.  Returns y in x's dtype, with a residual (y, h).
    Differentiable in x, weight, residual, from y and h (once; no forward mode)."""
    _check(x, weight, residual, eps, "rms_norm")
    y, h, _, _ = ops.rms_norm(x, residual, weight, eps)
    return y if residual is None else (y, h)


def rms_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
                   eps: float = 1e-6, out_dtype: torch.dtype = torch.float8_e4m3fn):
    """rms_norm with an 8-bit output for a product that follows: (codes,
    scales), with a residual (codes, scales, h).  codes: x's shape, out_dtype
    float8_e4m3fn or int8; scales: x's leading shape, fp32, y ~ codes * scale
    with scale = max(max |y| / qmax, 2^-126) of the row (qmax 448 / 127).  A row
    whose y holds a NaN or an infinity gets a scale that is not finite.  Not
    differentiable: inputs that require gradients are refused under grad mode."""
    _check(x, weight, residual, eps, "rms_norm_quant")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise ValueError("rms_norm_quant has no gradient: call it under torch.no_grad() or on detached tensors")
    codes, h, scales, _ = ops.rms_norm(x, residual, weight, eps, out_dtype=out_dtype)
    return (codes, scales) if residual is None else (codes, scales, h)


__all__ = ["rms_norm", "rms_norm_quant"]
