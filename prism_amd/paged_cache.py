"""Paged caches of keys and values, MI355X implementation (csrc/paged*.hip): the
sequences that a server holds share pages of 16 to 256 places, each sequence's listed
in a row of a page table; new tokens are appended with their keys' rotary positions
applied on the way, and attended over the pages.

Pages hold 16-bit elements, or 4 bits: the hardware's 4-bit float (a sign and one of 0,
0.5, 1, 1.5, 2, 3, 4, 6) with a power of two for each 32 channels, 4.25 bits an element,
1/3.76 of 16 bits' memory and reads.  The reference has no counterpart.

A decoding step of a layer, queries and keys as the projections give them:

    append_paged(k, v, k_cache, v_cache, page_table, kv_lens, freqs=freqs)
    o = flash_attn_paged(q, k_cache, v_cache, page_table, kv_lens)

with kv_lens counting the new tokens.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import ops

_PAGE_SIZES = (16, 32, 64, 128, 256)


def paged_cache(pages: int, page_size: int, heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16, bits: int = 16,
                device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """(k_cache, v_cache) of zeros: [pages, heads, page_size, head_dim] of dtype, or with
    bits=4 uint8 [pages, heads, page_size (head_dim / 2 + head_dim / 32)] (the codes of a
    page's places, then their scales)."""
    if page_size not in _PAGE_SIZES:
        raise ValueError(f"page_size {page_size} must be one of {_PAGE_SIZES}")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim {head_dim} unsupported by the MI355X kernels (64, 128)")
    if pages < 1 or heads < 1:
        raise ValueError(f"a cache needs pages and heads, got {pages} and {heads}")
    if bits not in (16, 4):
        raise ValueError(f"a cache holds 16 or 4 bits, not {bits}")
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"a cache holds bfloat16 or float16 (or 4 bits of them), not {dtype}")
    if bits == 16:
        return tuple(torch.zeros(pages, heads, page_size, head_dim, dtype=dtype, device=device) for _ in "kv")
    place = head_dim // 2 + head_dim // 32
    return tuple(torch.zeros(pages, heads, page_size * place, dtype=torch.uint8, device=device) for _ in "kv")


def _check_caches(name, k_cache, v_cache, D):
    """Heads of the caches, whose places hold D channels."""
    four = k_cache.dtype is torch.uint8
    if k_cache.dtype is not v_cache.dtype or not (four or k_cache.dtype in (torch.bfloat16, torch.float16)):
        raise TypeError(f"{name}: caches must be both bfloat16, float16 or uint8 (4 bits), got {k_cache.dtype} and {v_cache.dtype}")
    if D not in (64, 128):
        raise ValueError(f"{name}: head_dim {D} unsupported by the MI355X kernels (64, 128)")
    place, shape = D // 2 + D // 32, k_cache.shape
    if shape != v_cache.shape or len(shape) != (3 if four else 4) or shape[0] < 1 or shape[1] < 1 \
            or (shape[2] % place if four else shape[3] != D):
        want = "uint8 [pages, heads, page size (D / 2 + D / 32)]" if four else "[pages, heads, page size, D]"
        raise ValueError(f"{name}: caches must be {want} with D = {D}, got {tuple(shape)} and {tuple(v_cache.shape)}")
    size = shape[2] // place if four else shape[2]
    if size not in _PAGE_SIZES:
        raise ValueError(f"{name}: page size {size} must be one of {_PAGE_SIZES}")
    return shape[1]


def _check_table(name, page_table, lens):
    if page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[1] < 1:
        raise ValueError(f"{name}: page_table must be int32 [B, pages of a sequence], got {page_table.dtype} {tuple(page_table.shape)}")
    B = page_table.shape[0]
    if lens is not None and (lens.dtype is not torch.int32 or lens.shape != (B,)):
        raise ValueError(f"{name}: kv_lens must be int32 [{B}], got {lens.dtype} {tuple(lens.shape)}")
    return B


def _check_bounds(name, cu_seqlens, B):
    if cu_seqlens.dtype is not torch.int32 or cu_seqlens.shape != (B + 1,):
        raise ValueError(f"{name}: cu_seqlens must be int32 [{B + 1}], got {cu_seqlens.dtype} {tuple(cu_seqlens.shape)}")


def append_paged(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                 kv_lens: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None, freqs: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, interleaved: bool = True,
                 sections: Optional[Sequence[int]] = None, amplitude: float = 1.0) -> None:
    """Writes the keys and values of new tokens to their sequences' pages, in place.

    k, v: [T, Hk, D] bfloat16 or float16, D 64 or 128, any strides (best: adjacent channels):
    the new tokens of B sequences, T / B each, or rows cu_seqlens[b] to cu_seqlens[b + 1] - 1
    (int32 [B + 1] on the GPU, not decreasing; rows outside belong to none and are not
    stored).  kv_lens: int32 [B], the sequences' lengths with the new tokens, which are their
    last: token i of n stands at place kv_lens[b] - n + i.  page_table: int32 [B, width]; place
    p is place p % page_size of page page_table[b, p // page_size].  Tokens whose place is
    negative or beyond the table's width, or whose page is none of the cache's (-1, say), are
    not stored; other places are left as they are.  Sequences must not share a page that new
    tokens go to (else either's row, or pieces of both, are left).

    k_cache, v_cache: of paged_cache, or views with adjacent channels (and places, in 4 bits)
    and strides of whole 16 bytes, that share no memory; 16 bits: of k's dtype.  4 bits: 32 channels share the least
    power of two that keeps them within 6 times it (no smaller than 2^-126), and each is
    rounded to the nearest value (halves to the even code); 32 channels of which one is a NaN
    or an infinity are read as NaN.  Values whose level is beyond a type's largest are infinite
    where they are read in it (float16: from 57,344 on, next to 65,536; bfloat16: 2.98e38).

    freqs: float64 [pairs] (rotary_frequencies), or None for keys that are turned already:
    turns k as apply_rotary does, at positions (int32 or int64 [T], with sections [T, axes]) or
    by default at the tokens' places, rounded once to k's dtype (in float64 before, so that a
    value beside a border between two 4-bit codes falls on its own side: single results may
    differ from apply_rotary's by a step).  Not interleaved, 2 * pairs must be a multiple of
    16.  Not differentiable: k or v that require gradients are refused under grad mode."""
    if len(k.shape) != 3 or k.shape != v.shape:
        raise ValueError(f"append_paged: k and v must be [T, Hk, D], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype not in (torch.bfloat16, torch.float16) or v.dtype is not k.dtype:
        raise TypeError(f"append_paged: k and v must be both bfloat16 or both float16, got {k.dtype} and {v.dtype}")
    T, Hk, D = k.shape
    if _check_caches("append_paged", k_cache, v_cache, D) != Hk:
        raise ValueError(f"append_paged: {Hk} key heads do not fit caches of {k_cache.shape[1]}")
    if k_cache.dtype is not torch.uint8 and k_cache.dtype is not k.dtype:
        raise TypeError(f"append_paged: the caches must have k's dtype {k.dtype} (or 4 bits), got {k_cache.dtype}")
    B = _check_table("append_paged", page_table, kv_lens)
    if cu_seqlens is not None:
        _check_bounds("append_paged", cu_seqlens, B)
    elif T % B if B else T:
        raise ValueError(f"append_paged: {T} tokens do not share out over {B} sequences (cu_seqlens says how)")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (k, v, freqs)):
        raise ValueError("append_paged has no gradient: call it under torch.no_grad() or on detached tensors")
    axis_pairs = []
    if freqs is None:
        if positions is not None or sections is not None:
            raise ValueError("append_paged: positions and sections go with freqs")
    else:
        pairs = freqs.shape
        if freqs.dtype is not torch.float64:
            raise TypeError(f"append_paged: freqs must be float64 (far positions lose their place in less), got {freqs.dtype}")
        if len(pairs) != 1 or pairs[0] < 1 or 2 * pairs[0] > D:
            raise ValueError(f"append_paged: {tuple(pairs)} frequencies do not fit heads of {D} channels")
        if not interleaved and pairs[0] % 8:
            raise ValueError(f"append_paged: {2 * pairs[0]} turning channels, not interleaved, must be a multiple of 16")
        if sections is not None:
            if positions is None:
                raise ValueError("append_paged: sections need positions, one entry per axis")
            if any(int(n) < 2 or int(n) % 2 for n in sections) or sum(int(n) for n in sections) != 2 * pairs[0]:
                raise ValueError(f"append_paged: sections {list(sections)} must be even and sum to {2 * pairs[0]}")
            axis_pairs = [int(n) // 2 for n in sections]
        if positions is not None and positions.shape != ((T,) if sections is None else (T, len(axis_pairs))):
            raise ValueError(f"append_paged: positions must be [{T}]{' with one entry per axis' if axis_pairs else ''}, "
                             f"got {tuple(positions.shape)}")
    ops.paged_append(k, v, k_cache, v_cache, page_table, kv_lens, cu_seqlens, freqs, positions, axis_pairs, interleaved, amplitude)


def gather_paged(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor, total: int, *,
                 head_dim: Optional[int] = None, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [total, heads, D], dense: places 0 .. n_b - 1 of every sequence, n_b =
    cu_seqlens[b + 1] - cu_seqlens[b], one sequence behind the other (rows of no sequence, and
    places without a page, are 0): what flash_attn_packed takes as its keys for the next part
    of prompts whose first part is cached.  head_dim: D, needed for 4-bit caches; dtype:
    bfloat16 (default) or float16 of what 4 bits hold (in bfloat16 exactly); of 16-bit caches
    theirs."""
    four = k_cache.dtype is torch.uint8
    if head_dim is None:
        if four:
            raise ValueError("gather_paged: a 4-bit cache needs head_dim")
        head_dim = k_cache.shape[-1]
    heads = _check_caches("gather_paged", k_cache, v_cache, head_dim)
    want = dtype if dtype is not None else torch.bfloat16 if four else k_cache.dtype
    if want not in (torch.bfloat16, torch.float16) or (not four and want is not k_cache.dtype):
        raise TypeError(f"gather_paged: dtype {dtype} of a {k_cache.dtype} cache")
    B = _check_table("gather_paged", page_table, None)
    _check_bounds("gather_paged", cu_seqlens, B)
    if total < 0:
        raise ValueError(f"gather_paged: total must not be negative, got {total}")
    return ops.paged_gather(k_cache, v_cache, page_table, cu_seqlens, total, heads, head_dim, want is torch.float16)


def flash_attn_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                     kv_lens: torch.Tensor, *, sm_scale: Optional[float] = None, return_lse: bool = False):
    """softmax(sm_scale q k^T) v of new tokens over a paged cache.

    q: [T, Hq, D] bfloat16 or float16, D 64 or 128, any strides (best: adjacent channels): T /
    B tokens of each of B sequences, the last of the sequence's kv_lens[b] (int32 [B]), which
    are in the cache already: token i of n sees places j <= kv_lens[b] - n + i.  Hq a multiple of
    the caches' heads (query heads h * Hq / Hk .. share key head h).  k_cache, v_cache,
    page_table: as for append_paged; 16 bits: of q's dtype.  Lengths beyond the table's width are
    cut to it.  Places beyond a sequence's length may hold anything; places whose table entry
    is no page (-1, say) are not seen.  Tokens that see nothing give 0.  Made for few tokens (up
    to 32 rows of tokens x Hq / Hk share one read of the cache); for more, gather_paged and
    flash_attn_packed.  sm_scale (positive) defaults to D^-1/2.  A NaN or an infinity in a key
    or value reaches the tokens that see it and no others (4 bits: as NaN, a value's where the
    key's weight is not below 2^-126 of the largest's).  4 bits: values of 2^100 and more may
    become infinite in the sums.

    Returns o, of q's shape (and layout, where q is dense), with return_lse (o, lse): lse [Hq,
    T] float32, the natural log of the sum of exponentials of the scaled scores, -inf where
    nothing is seen.  Not differentiable: q that requires gradients is refused under grad
    mode."""
    if len(q.shape) != 3:
        raise ValueError(f"flash_attn_paged: q must be [T, Hq, D], got {tuple(q.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"flash_attn_paged: q must be bfloat16 or float16, got {q.dtype}")
    T, Hq, D = q.shape
    Hk = _check_caches("flash_attn_paged", k_cache, v_cache, D)
    if Hq < Hk or Hq % Hk:
        raise ValueError(f"{Hq} query heads do not share {Hk} key heads evenly")
    if k_cache.dtype is not torch.uint8 and k_cache.dtype is not q.dtype:
        raise TypeError(f"flash_attn_paged: the caches must have q's dtype {q.dtype} (or 4 bits), got {k_cache.dtype}")
    B = _check_table("flash_attn_paged", page_table, kv_lens)
    if T % B if B else T:
        raise ValueError(f"flash_attn_paged: {T} queries do not share out over {B} sequences")
    if torch.is_grad_enabled() and q.requires_grad:
        raise ValueError("flash_attn_paged has no gradient: call it under torch.no_grad() or on detached tensors")
    sm_scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    if not 0 < sm_scale < float("inf"):
        raise ValueError(f"sm_scale must be positive and finite, got {sm_scale}")
    o, lse = ops.paged_fwd(q, k_cache, v_cache, page_table, kv_lens, Hk, sm_scale, return_lse)
    return (o, lse) if return_lse else o


__all__ = ["paged_cache", "append_paged", "gather_paged", "flash_attn_paged"]
