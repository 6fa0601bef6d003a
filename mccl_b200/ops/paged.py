"""A paged key-value cache's operators: tokens into its pages, attention of new tokens over it, copies of its pages.

Keys and values of a layer are ``[pages, kv_heads, page_size, head_dim]`` (any strides with a contiguous head_dim that are multiples of 8
elements); a page table, int32 ``[sequences, width]``, names the pages of every sequence in order.  All sizes that change from token to token
are on the device (positions, lengths, the table), so a step can be captured in a CUDA graph.  bf16 and fp16; forward only.

CUDA tensors run this package's kernels; CPU tensors run the plain forms below (tests without a GPU).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .. import _C


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, positions: torch.Tensor,
                 rows: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None, rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """Writes keys and values of new tokens, ``[tokens, kv_heads, head_dim]`` each, into their pages.

    Token t is at ``positions[t]`` (int32) of the sequence in row ``rows[t]`` of the table (int32; without `rows`, row t).  A token with a
    negative position, or whose row, position or page lies outside the table or the cache, writes nothing.  No two tokens may have the same place.

    rope: (cos, sin), fp32 ``[positions, head_dim / 2]``: keys are rotated on the way, and so is `q` ``[tokens, heads, head_dim]``, which is
    returned as a new tensor (zero for a token that writes nothing; a position beyond the tables counts as outside).  Without rope None is returned."""
    cos, sin = rope if rope is not None else (None, None)
    if k.is_cuda:
        return _C.paged_append(k, v, k_pages, v_pages, page_table, positions, rows, q, cos, sin)
    if q is not None and rope is None:
        raise RuntimeError("paged_append: q is only taken to be rotated, and there are no rotation tables")
    page = k_pages.shape[2]
    at = positions.long()
    row = torch.arange(k.shape[0]) if rows is None else rows.long()
    good = (at >= 0) & (row >= 0) & (row < page_table.shape[0]) & (at // page < page_table.shape[1])
    if rope is not None:
        good &= at < cos.shape[0]
    index = torch.full_like(at, -1)
    index[good] = page_table[row[good], at[good] // page].long()
    good &= (index >= 0) & (index < k_pages.shape[0])

    def rotate(x):
        c, s = cos[at.clamp(0, cos.shape[0] - 1)][:, None], sin[at.clamp(0, cos.shape[0] - 1)][:, None]
        a, b = x[..., 0::2].float(), x[..., 1::2].float()
        return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2).to(x.dtype)

    keys = k if rope is None else rotate(k)
    k_pages[index[good], :, at[good] % page] = keys[good]
    v_pages[index[good], :, at[good] % page] = v[good]
    return None if q is None else torch.where(good[:, None, None], rotate(q), 0)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                    scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0, return_lse: bool = False):
    """Attention of one new token per sequence, ``q`` ``[sequences, heads, head_dim]``, over the first ``lengths[b]`` positions (int32, the new
    token's own among them) of each: softmax(scale q.K) V, ``[sequences, heads, head_dim]``; scale defaults to ``head_dim ** -0.5``.

    heads is a multiple of the cache's kv_heads: neighbouring query heads share keys and values.  With `window`, only the last `window`
    positions and the first `sinks` are seen; pages without a visible position are not looked at (their table entries may be -1).
    A sequence of length zero gives zeros.  A length beyond the table's row counts as the row's; a visible position whose page
    lies outside the cache is left out (NaN where none is left).  What lies at positions that are not seen may be anything; an infinite value at
    one that is seen makes its column NaN (weights are kept in two parts, of which one may be zero).

    return_lse: also the logarithm of the sum of exponentials, fp32 ``[sequences, heads]`` (-inf for an empty sequence), with which parts of
    a longer attention can be joined."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if window is None:
        if sinks:
            raise RuntimeError("paged_attention: sinks without a window")
    elif window < 1:
        raise RuntimeError(f"paged_attention: window must be positive, got {window}")
    if q.is_cuda:
        o, lse = _C.paged_attention(q, k_pages, v_pages, page_table, lengths, scale, 0 if window is None else window, sinks, return_lse)
        return (o, lse) if return_lse else o
    batch, heads, dim = q.shape
    kv_heads, page = k_pages.shape[1], k_pages.shape[2]
    out, lse = torch.zeros_like(q, memory_format=torch.contiguous_format), torch.full((batch, heads), -math.inf)
    for b in range(batch):
        length = min(max(int(lengths[b]), 0), page_table.shape[1] * page)
        j = torch.arange(length)
        if window is not None:
            j = j[(j >= length - window) | (j < sinks)]
        index = page_table[b, j // page].long()
        j, index = (t[(index >= 0) & (index < k_pages.shape[0])] for t in (j, index))
        if length == 0:
            continue
        k, v = (t[index, :, j % page].float().repeat_interleave(heads // kv_heads, dim=1) for t in (k_pages, v_pages))
        score = torch.einsum("hd,jhd->hj", q[b].float(), k) * scale
        lse[b] = torch.logsumexp(score, dim=-1) if len(j) else -math.inf
        out[b] = torch.einsum("hj,jhd->hd", torch.softmax(score, dim=-1), v).to(q.dtype) if len(j) else math.nan
    return (out, lse) if return_lse else out


def copy_pages(pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, dim: int = 0) -> torch.Tensor:
    """``pages[..., dst[i], ...] = pages[..., src[i], ...]`` along `dim` for all i, in place, in one kernel; returns `pages`.  src, dst: int32.

    What follows `dim` has to be contiguous (a page), what precedes it (layers, keys and values) evenly spaced.  A page may be named once
    among dst, and not as the source of another copy; a pair with an index outside the cache is skipped.  Any dtype."""
    if pages.is_cuda:
        return _C.copy_pages(pages, src, dst, dim)
    n = pages.shape[dim]
    good = (src >= 0) & (src < n) & (dst >= 0) & (dst < n)
    return pages.index_copy_(dim, dst[good].long(), pages.index_select(dim, src[good].long()))
