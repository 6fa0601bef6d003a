"""Linear layers with 4-bit weights: a code of 0..15 per weight, a scale and a zero point per row and group of columns.

``w[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group])``.  CUDA tensors run this package's kernels; CPU tensors run the
plain form (tests without a GPU).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F

from .. import _C

GROUPS = (32, 64, 128, 256)


class W4Weight:
    """A weight ``[n, k]`` in 4 bits, laid out once for the kernels.

    ``codes``: uint8 ``[ceil(n / 16), ceil(k / 64), 32, 16]``, tiles of 16 rows and 64 columns.  Word s of lane 4 g + t has of columns 16 s .. 16 s + 15
    the codes of rows g and g + 8 in columns 2 t, 2 t + 1, 2 t + 8 and 2 t + 9: what a lane holds of the left operand of a 16 x 8 x 16 product.
    ``params``: int32 ``[ceil(n / 16), k / group, 8, 2]``, rows g and g + 8: the scale's bf16 bits, above them those of 128 + zero."""

    def __init__(self, codes: torch.Tensor, params: torch.Tensor, n: int, k: int, group: int):
        self.codes, self.params, self.n, self.k, self.group = codes, params, n, k, group

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.n, self.k))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.params.numel()

    def to(self, device) -> "W4Weight":
        return W4Weight(self.codes.to(device), self.params.to(device), self.n, self.k, self.group)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None) -> "W4Weight":
        """codes: uint8 ``[n, k]``, 0..15; scales ``[n, k / group]``, kept as bf16; zeros: uint8 of the same shape, 0..15 (None: 8)."""
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise RuntimeError("W4Weight: codes must be uint8 [n, k]")
        n, k = codes.shape
        if scales.dim() != 2 or scales.shape[0] != n or scales.shape[1] == 0 or k % scales.shape[1] or not scales.is_floating_point():
            raise RuntimeError(f"W4Weight: scales must be floating-point [{n}, groups] with groups that divide {k}")
        group, groups = k // scales.shape[1], scales.shape[1]
        if group not in GROUPS:
            raise RuntimeError(f"W4Weight: groups of {group} columns; {', '.join(map(str, GROUPS))} are supported")
        if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != torch.uint8):
            raise RuntimeError("W4Weight: zeros must be uint8 of the scales' shape")
        if any(t is not None and t.device != codes.device for t in (scales, zeros)):
            raise RuntimeError("W4Weight: codes, scales and zeros on different devices")
        if codes.is_cuda:
            packed, params, bad = _C.w4_pack(codes.contiguous(), scales.to(torch.bfloat16).contiguous(), None if zeros is None else zeros.contiguous())
        else:
            bad = codes.numel() and (int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15))
        if bad:
            raise RuntimeError("W4Weight: codes and zeros are numbers from 0 to 15")
        if codes.is_cuda:
            return cls(packed, params, n, k, group)
        tiles, chunks = -(-n // 16), -(-k // 64)
        padded = F.pad(codes, (0, chunks * 64 - k, 0, tiles * 16 - n)) if (n % 16 or k % 64) else codes
        # rows: 8 r + g; columns of a chunk: 16 s + 8 q + 2 t + e.  Nibble 4 e + 2 q + r of word s.
        c = padded.reshape(tiles, 2, 8, chunks, 4, 2, 4, 2)
        packed = c[:, 0] | (c[:, 1] << 4)                                       # [tile, g, chunk, s, q, t, e]
        packed = packed.permute(0, 2, 1, 5, 3, 6, 4).reshape(tiles, chunks, 32, 16).contiguous()
        scale = F.pad(scales.to(torch.bfloat16), (0, 0, 0, tiles * 16 - n)).view(torch.int16).to(torch.int32) & 0xffff
        zero = F.pad(torch.full_like(scale[:n], 8) if zeros is None else zeros.to(torch.int32), (0, 0, 0, tiles * 16 - n))
        params = scale | ((zero + 0x4300) << 16)                                # bf16 128 is 0x4300, and its last bit is worth one
        params = params.view(tiles, 2, 8, groups).permute(0, 3, 2, 1).contiguous()
        return cls(packed, params, n, k, group)

    def dequantize(self) -> torch.Tensor:
        """The weight as bf16 ``[n, k]``."""
        if self.codes.is_cuda:
            return _C.w4_dequantize(self.codes, self.params, self.n, self.k, self.group)
        return self._plain().to(torch.bfloat16)

    def _plain(self) -> torch.Tensor:
        tiles, chunks = self.codes.shape[:2]
        b = self.codes.view(tiles, chunks, 8, 4, 4, 2, 2)                       # [tile, chunk, g, t, s, e, q]
        c = torch.stack((b & 15, b >> 4), dim=1)                                # [tile, r, chunk, g, t, s, e, q]
        c = c.permute(0, 1, 3, 2, 5, 7, 4, 6).reshape(tiles * 16, chunks * 64)[: self.n, : self.k]
        p = self.params.permute(0, 3, 2, 1).reshape(tiles * 16, -1)[: self.n]
        zero = ((p >> 16) & 0xffff) - 0x4300
        scale = (p & 0xffff).to(torch.int16).view(torch.bfloat16).float() if p.numel() else p.float()
        w = (c.view(self.n, -1, self.group).float() - zero[..., None].float()) * scale[..., None]
        return w.view(self.n, self.k)


def quantize_w4(weight: torch.Tensor, group: int = 128) -> W4Weight:
    """4-bit weight of ``[n, k]``: for each group of columns of a row the scale and zero point that span its values (and zero)."""
    if weight.dim() != 2 or weight.shape[1] % group or group not in GROUPS:
        raise RuntimeError(f"quantize_w4: a weight [n, k] with k a multiple of the group, one of {GROUPS}; got {tuple(weight.shape)} and {group}")
    n, k = weight.shape
    w = weight.detach().float().view(n, k // group, group)
    low, high = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
    scale = ((high - low) / 15.0).to(torch.bfloat16).float()
    if not bool(torch.isfinite(scale).all()):
        raise RuntimeError("quantize_w4: weights that are not finite, or that no scale spans")
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = (-low / scale).round().clamp(0, 15)
    codes = (w / scale[..., None]).round().add(zero[..., None]).clamp(0, 15).to(torch.uint8).view(n, k)
    return W4Weight.from_codes(codes, scale, zero.to(torch.uint8))


def linear_w4(x: torch.Tensor, weight: W4Weight, bias: Optional[torch.Tensor] = None, act: str = "none", residual: Optional[torch.Tensor] = None):
    """act(x @ W^T + b) + residual for x bf16 ``[..., k]``; bias fp32 ``[n]``; act "none" or "gelu".  Forward only.

    With up to 16 rows of x (fewer where 256 bytes per row and 128 columns pass 128 KB) codes are multiplied as whole numbers and scaled in fp32, so that
    nothing but x and the result is rounded; with more rows ``scale * (code - zero)`` is rounded to bf16 first, as :meth:`W4Weight.dequantize` has it.
    Sums are fp32 either way, and added in an order that depends on the sizes only."""
    gelu = act == "gelu"
    if not gelu and act != "none":
        raise RuntimeError(f"linear_w4: unknown activation '{act}'")
    if x.is_cuda:
        return _C.w4_linear(x, weight.codes, weight.params, weight.n, weight.k, weight.group, bias, gelu, residual)
    y = F.linear(x.float(), weight._plain(), None if bias is None else bias.float())
    if act == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return (y if residual is None else y + residual.float()).to(x.dtype)
