"""4-bit weight packing for ``linear_w4``: laid out once, at load time.

A weight stands for ``(code - zero) * scale`` with a code of 0 to 15 and one scale,
and one zero point (8 unless given), per group of 32, 64 or 128 weights along the
reduction axis.  ``pack_w4`` brings codes ``[N, K]`` (a checkpoint's, unpacked from
its own order) into the order in which the kernel reads them; ``quantize_w4`` makes
codes, scales and zero points from weights.

Rows are padded to whole blocks of 128 codes, 64 bytes: as little-endian 32-bit
words, word ``4 t + s`` of a block holds the codes of ``k = 32 s + 8 t + 0..7`` of
it, ``k = 2 i`` in bits ``4 i``, ``k = 2 i + 1`` in bits ``16 + 4 i``.
"""
from __future__ import annotations

import torch

BLOCK = 128
GROUPS = (32, 64, 128)


def pack_w4(codes: torch.Tensor) -> torch.Tensor:
    """Codes [N, K] of 0 to 15 -> uint8 [N, ceil(K / 128) * 64]."""
    if codes.dim() != 2:
        raise ValueError("codes must be [N, K]")
    N, K = codes.shape
    blocks = -(-K // BLOCK)
    c = torch.zeros(N, blocks * BLOCK, dtype=torch.uint8, device=codes.device)
    c[:, :K] = codes
    if bool((c > 15).any()) or bool((c[:, :K] != codes).any()):
        raise ValueError("codes must be whole numbers, 0 to 15")
    c = c.view(N, blocks, 4, 4, 4, 2).permute(0, 1, 3, 2, 5, 4).reshape(N, blocks * 64, 2)  # block, t, s, odd, pair
    return c[..., 0] | c[..., 1] << 4


def unpack_w4(packed: torch.Tensor, K: int) -> torch.Tensor:
    """The codes [N, K] of `packed`."""
    N, blocks = packed.shape[0], packed.shape[1] // 64
    c = torch.stack([packed & 15, packed >> 4], dim=-1).view(N, blocks, 4, 4, 2, 4)  # block, t, s, odd, pair
    return c.permute(0, 1, 3, 2, 5, 4).reshape(N, blocks * BLOCK)[:, :K]


def quantize_w4(w: torch.Tensor, group: int = 128, zero_points: bool = False, dtype: torch.dtype = torch.bfloat16):
    """(packed, scale [N, K / group] of `dtype`, zero uint8 or None) of weights [N, K].

    Without zero points the codes 1 to 15 span a group's largest magnitude evenly
    around 8; with them 0 to 15 span its range, 0 included.  Codes are the nearest
    to the weights for the scale as it is stored.  Weights must be finite, and a
    group's scale within `dtype`.
    """
    if w.dim() != 2 or group not in GROUPS or w.shape[1] % group:
        raise ValueError("w must be [N, K] with K a multiple of group (32, 64 or 128)")
    N, K = w.shape
    g = w.float().view(N, K // group, group)
    if zero_points:
        lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
        scale = ((hi - lo) / 15).to(dtype)
    else:
        scale = (g.abs().amax(-1) / 7).to(dtype)
    if not bool(torch.isfinite(scale).all()):
        raise ValueError(f"weights must be finite, and a group's scale within {dtype}")
    step = torch.where(scale.float() > 0, scale.float(), 1.0)[..., None]
    zero = torch.round(-lo[..., None] / step).clamp(0, 15) if zero_points else torch.full_like(step, 8.0)
    codes = (torch.round(g / step) + zero).clamp(0 if zero_points else 1, 15).to(torch.uint8)
    return pack_w4(codes.view(N, K)), scale, zero[..., 0].to(torch.uint8) if zero_points else None


def dequantize_w4(packed: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None, K: int) -> torch.Tensor:
    """float32 weights [N, K]."""
    N, groups = scale.shape
    c = unpack_w4(packed, K).float().view(N, groups, K // groups)
    z = zero.float()[..., None] if zero is not None else 8.0
    return ((c - z) * scale.float()[..., None]).view(N, K)
