"""8-bit rows and their projections from the definition, in 64 bits (test infrastructure only).

A row of `width` columns is e4m3 values with one power of two per block of 128 columns. The
functions here work on what the bits stand for: float64 tensors of values and int64 tensors of
biased exponents (the power is 2^(s - 127)).
"""

from __future__ import annotations

from typing import Tuple

import torch
from torch import Tensor

BLOCK = 128
LARGEST = 448.0


def blocks(width: int) -> int:
    return -(-width // BLOCK)


def padded_blocks(y: Tensor) -> Tensor:
    """[rows, width] as [rows, blocks, 128], zeros past the columns."""
    rows, width = y.shape
    out = torch.zeros((rows, blocks(width) * BLOCK), dtype=y.dtype)
    out[:, :width] = y
    return out.view(rows, -1, BLOCK)


def largest(y: Tensor) -> Tensor:
    """The largest finite magnitude of each block."""
    magnitude = padded_blocks(y).abs()
    return torch.where(torch.isfinite(magnitude), magnitude, torch.zeros_like(magnitude)).amax(-1)


def exponents(most: Tensor) -> Tensor:
    """Biased exponents of the smallest powers of two with 448 * 2^(s - 127) >= most, at least 1."""
    found = torch.ones(most.shape, dtype=torch.int64)
    for s in range(1, 255):
        found = torch.where(most > LARGEST * 2.0 ** (s - 127), s + 1, found)
    return found


def step(v: Tensor) -> Tensor:
    """The distance of e4m3 neighbours around |v| (the wider one at a power of two)."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6))) - 3)


def round_e4m3(v: Tensor) -> Tensor:
    """To the nearest e4m3, ties to the even neighbour; |v| <= 448, infinities and NaN to NaN."""
    out = torch.round(v / step(v)) * step(v)
    return torch.where(torch.isfinite(v), out, torch.full_like(v, float("nan")))


def spread(s: Tensor, width: int) -> Tensor:
    """2^(s - 127) of each column."""
    return torch.exp2(s.double() - 127.0).repeat_interleave(BLOCK, dim=1)[:, :width]


def round_rows(y: Tensor) -> Tuple[Tensor, Tensor]:
    """float64 rows to (e4m3 values, biased exponents)."""
    s = exponents(largest(y))
    return round_e4m3(y / spread(s, y.shape[1])), s


def stands_for(values: Tensor, s: Tensor) -> Tensor:
    """What 8-bit rows stand for: values (any float tensor) times their blocks' powers."""
    return values.double() * spread(s[:, : blocks(values.shape[1])], values.shape[1])


def add_rms_norm(hidden: Tensor, delta: Tensor | None, weight: Tensor, eps: float) -> Tuple[Tensor, Tensor]:
    """(residual sum rounded to fp16, norm before its rounding) of fp16 rows; delta fp16 or None."""
    total = hidden.double() if delta is None else (hidden.double() + delta.double()).half().double()
    return total, total / torch.sqrt((total * total).mean(-1, keepdim=True) + eps) * weight.double()


def split_columns(k: int, splits: int) -> list[int]:
    """Where the K splits begin, and the end."""
    return [min(k, BLOCK * (s * blocks(k) // splits)) for s in range(splits + 1)]


def swiglu(y: Tensor) -> Tensor:
    gate, up = y.chunk(2, dim=1)
    return gate / (1.0 + torch.exp(-gate)) * up
