"""Whole prompts and packed texts: causal attention of texts of different lengths that lie one behind the other, without padding between them, and
rotary positions of any tokens.

Queries, keys and values are ``[tokens, heads, head_dim]``; ``offsets``, int32 ``[texts + 1]`` on the device, says where each text begins (and the
last one ends).  Nothing of a call depends on numbers the host would have to wait for, so it can be captured in a CUDA graph.

CUDA tensors run this package's kernels; CPU tensors run the plain forms below (tests without a GPU).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .. import _C


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, k_offsets: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                     window: Optional[int] = None, sinks: int = 0, return_lse: bool = False):
    """Causal attention within each of the texts: softmax(scale q.K) V for q ``[tokens, heads, head_dim]`` and k, v ``[tokens, kv_heads, head_dim]``;
    scale defaults to ``head_dim ** -0.5``.  bf16 and fp16, head dimensions of up to 128 (multiples of 8); gradients of q, k and v in bf16.

    Text s has the tokens ``offsets[s]`` to ``offsets[s + 1] - 1``; offsets do not decrease, a text may be empty.  With `k_offsets` its keys are
    ``k_offsets[s]`` to ``k_offsets[s + 1] - 1`` instead: those in front of its queries are from before (a prompt that goes on behind what a cache
    holds), the last query stands at the last key.  heads is a multiple of kv_heads: neighbouring query heads share keys and values.
    With `window`, only the last `window` positions and the first `sinks` of the text are seen.

    Rows of no text, and queries that see nothing (more queries than keys), give zeros, and zero gradients.  What lies at positions that a query does not
    see has no influence on its result, whatever it is; an infinite or NaN value at one that is seen makes its column infinite or NaN.  In the gradients
    such numbers may reach other positions of the same text, but no other text.

    For the gradients a call keeps q, k and v, its result with what its rounding left (so twice the result's memory), and the logarithms below.

    return_lse: also the logarithm of the sum of exponentials, fp32 ``[tokens, heads]`` (-inf where nothing is seen; no gradient)."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if not 0 < scale < 2e38:   # (times log2 e it must be a number of 32 bits: beyond 2.36e38 every result was NaN)
        raise RuntimeError(f"packed_attention: scale must be a positive number below 2e38, got {scale}")
    if window is None:
        if sinks:
            raise RuntimeError("packed_attention: sinks without a window")
    elif window < 1:
        raise RuntimeError(f"packed_attention: window must be positive, got {window}")
    if q.is_cuda:
        o, lse = _C.packed_attention(q, k, v, offsets, k_offsets, scale, 0 if window is None else window, sinks, return_lse)
        return (o, lse) if return_lse else o
    starts = offsets.tolist()
    key_starts = starts if k_offsets is None else k_offsets.tolist()
    group = q.shape[1] // k.shape[1]
    parts, sums, at = [], [], 0
    nothing = q.new_zeros((0, *q.shape[1:])), torch.zeros(0, q.shape[1])

    def rows_without(n):
        parts.append(q.new_zeros((n, *q.shape[1:])))
        sums.append(torch.full((n, q.shape[1]), -math.inf))

    for first, last, key, key_end in zip(starts, starts[1:], key_starts, key_starts[1:]):
        rows_without(first - at)
        n, m, at = last - first, key_end - key, last
        blind = min(n, max(0, n - m))   # these stand in front of the first key
        rows_without(blind)
        if n == blind:
            continue
        i, j = torch.arange(m - (n - blind), m)[:, None], torch.arange(m)[None]
        seen = j <= i
        if window is not None:
            seen = seen & ((j > i - window) | (j < sinks))
        qq, kk, vv = q[first + blind:last].float(), *(t[key:key_end].float().repeat_interleave(group, dim=1) for t in (k, v))
        score = torch.where(seen, torch.einsum("ihd,jhd->hij", qq, kk) * scale, -math.inf)
        sums.append(torch.logsumexp(score, -1).t())
        parts.append(torch.einsum("hij,jhd->ihd", torch.softmax(score, -1), vv).to(q.dtype))
    rows_without(q.shape[0] - at)
    o = torch.cat([nothing[0], *parts])
    return (o, torch.cat([nothing[1], *sums]).detach()) if return_lse else o


def rotary(q: torch.Tensor, k: Optional[torch.Tensor] = None, *, rope: Tuple[torch.Tensor, torch.Tensor], positions: Optional[torch.Tensor] = None, layout: str = "interleaved"):
    """Queries and keys turned by their positions: new tensors (q, k), or q alone without `k`.  q ``[tokens, heads, head_dim]``, k of the same tokens; bf16 or
    fp16, differentiable.

    rope: (cos, sin), fp32 ``[positions, pairs]`` (:func:`rotary_tables`).  The first ``2 * pairs`` elements of each head are turned, what is behind them stays.
    Pairs are neighbours in the layout "interleaved" (that of :func:`paged_append` and of this package's models) and `pairs` apart in the layout "half".
    positions: int32 ``[tokens]`` (without it, token t stands at t).  A token whose position lies outside the tables becomes zeros."""
    if layout not in ("interleaved", "half"):
        raise RuntimeError(f"rotary: layouts are 'interleaved' and 'half', not '{layout}'")
    cos, sin = rope
    if q.is_cuda:
        a, b = _C.rotary(q, k, cos, sin, positions, layout == "half")
        return a if k is None else (a, b)
    pairs = cos.shape[1]
    at = torch.arange(q.shape[0]) if positions is None else positions.long()
    inside = (at >= 0) & (at < cos.shape[0])
    c, s = (t[at.clamp(0, max(0, cos.shape[0] - 1))][:, None] if cos.shape[0] else t.new_zeros(len(at), 1, pairs) for t in (cos, sin))

    def turn(x):
        part = x[..., :2 * pairs].float()
        a, b = (part[..., 0::2], part[..., 1::2]) if layout == "interleaved" else (part[..., :pairs], part[..., pairs:])
        a, b = a * c - b * s, a * s + b * c
        part = torch.stack((a, b), dim=-1).flatten(-2) if layout == "interleaved" else torch.cat((a, b), dim=-1)
        return torch.where(inside[:, None, None], torch.cat((part.to(x.dtype), x[..., 2 * pairs:]), dim=-1), 0)

    return turn(q) if k is None else (turn(q), turn(k))


def rotary_tables(positions: int, dim: int, *, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0, original: Optional[int] = None,
                  magnitude: float = 1.0, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 ``[positions, dim / 2]``, of position times ``theta ** (-2 i / dim)``, from angles in 64 bits (far positions keep their angle).

    scaling, for texts `factor` times longer than a model was trained on:
      "linear"  all angles are divided by the factor
      "base"    theta grows so that the slowest pair's angle is divided by the factor and the fastest stays
      "bands"   pairs that turn 32 times or more within `original` positions stay, those that turn once or less are divided by the factor, those in between go
                from one to the other evenly with the number of turns
    magnitude: both tables times this."""
    if positions < 0 or dim < 2 or dim % 2 or not theta > 0 or not factor > 0:
        raise RuntimeError(f"rotary_tables: no tables of {positions} positions, {dim} elements, theta {theta} and factor {factor}")
    step = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    if scaling == "base":
        if dim < 4:
            raise RuntimeError("rotary_tables: one pair has no slowest and fastest")
        theta = theta * factor ** (dim / (dim - 2))
    speed = theta ** -step
    if scaling == "linear":
        speed = speed / factor
    elif scaling == "bands":
        if original is None or original < 1:
            raise RuntimeError("rotary_tables: scaling 'bands' needs the original number of positions")
        share = ((original * speed / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)   # how much of the pair stays as it was
        speed = speed * share + speed / factor * (1.0 - share)
    elif scaling not in (None, "base"):
        raise RuntimeError(f"rotary_tables: scalings are 'linear', 'base' and 'bands', not '{scaling}'")
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device=device), speed.to(device))
    return (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
