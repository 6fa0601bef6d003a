"""The choice of tokens from logits, by given random numbers.

CUDA tensors run this package's kernel; CPU tensors run the plain form below (tests without a GPU).
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _C

Setting = Union[float, torch.Tensor, None]


def sample(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Setting = 1.0, top_k: Union[int, torch.Tensor, None] = None, top_p: Setting = None,
           min_p: Setting = None) -> torch.Tensor:
    """A token for each row of logits ``[rows, vocab]`` (bf16, fp16 or fp32, up to 2^20 tokens), int64 ``[rows]``, for uniform numbers from 0 up to 1, fp32 or fp64
    ``[rows]``: the same numbers give the same tokens.  Nothing waits for the host; a call can be captured in a CUDA graph.

    With w = exp((logit - the row's highest) / temperature), one after the other:
      top_k  keeps the `top_k` likeliest tokens (of equal ones those with the lowest numbers; 0 or None: all)
      top_p  of these keeps the fewest likeliest whose w add up to `top_p` of the sum over these (1 or None: all; at least one stays)
      min_p  of these keeps those whose w is `min_p` or more (0 or None: all)
    The token is the lowest one at which the running sum of the kept w exceeds its row's uniform number times their whole sum.  Temperature 0: the likeliest
    token.  Each setting is a number, or one per row (fp32 ``[rows]``; int32 for top_k); numbers count as fp32.  A w is off by less
    than 2^-36 of itself and 2^-44, sums of them are exact.

    A row with a NaN or +inf, or with nothing finite, gives -1, and so does one whose temperature is negative or NaN."""
    settings = (temperature, 0 if top_k is None else top_k, 1.0 if top_p is None else top_p, 0.0 if min_p is None else min_p)
    if logits.is_cuda:
        return _C.sample(logits, uniform, *settings)
    rows, vocab = logits.shape
    for name, value, high in zip(("temperature", "top_k", "top_p", "min_p"), settings, (3.4e38, 2 ** 31 - 1, 1.0, 1.0)):
        if not torch.is_tensor(value) and not (0 <= value <= high and (name != "top_k" or value == int(value))):
            raise RuntimeError(f"sample({name}): {value} is out of range")
    t, k, p, low = (torch.as_tensor(v, dtype=torch.float32).double().expand(rows)[:, None] for v in settings)
    x = logits.double()
    high = x.amax(-1, keepdim=True)
    usable = torch.isfinite(high[:, 0]) & ~torch.isnan(x).any(-1) & (t[:, 0] >= 0)
    weight = torch.exp((x - high) / torch.where(t > 0, t, 1.0)).nan_to_num(0.0)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    ordered, rank = weight.gather(1, order), torch.arange(vocab)
    kept = (k <= 0) | (rank < k)
    sums = torch.cumsum(torch.where(kept, ordered, 0.0), -1)
    kept = kept & (~(p < 1) | (rank == 0) | (sums - ordered < p * sums[:, -1:]))
    kept = kept & ~(ordered < low.clamp(max=1.0))
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    sums = torch.cumsum(torch.where(kept, weight, 0.0), -1)
    u = uniform.double()[:, None]
    passed = kept & (weight > 0) & ((sums > u * sums[:, -1:]) | (sums == sums[:, -1:]))
    chosen = torch.where(t > 0, passed, x == high).int().argmax(-1)
    return torch.where(usable, chosen, -1)
