"""The 4-bit KV pool from its definition, in 64 bits, an element at a time (test infrastructure only).

A row x (64 values of one token, kv head and kind) is lo = min(x), s = the smallest fp16 with
15 s >= max(x) - lo, and levels n = round((x - lo) / s), half to even, for the values lo + s n; (NaN, 0) for
a row with an infinity or NaN. The differences are rounded to fp32 (they are exact but in rows whose magnitudes
span more than 2^13), the rest is exact; a lo of zero is +0.
"""

from __future__ import annotations

from typing import Sequence, Tuple

import numpy as np

UNIT, HEADS, DIM, SLOTS, LAYERS = 1152, 4, 64, 16, 22

_FP16 = np.arange(0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)  # every finite fp16 >= 0, rising


def quantize(x: np.ndarray) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Rows float16 [..., 64] as (levels int64 [..., 64], lo float16 [...], s float16 [...])."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        y = x.astype(np.float32)
        fine = np.isfinite(y).all(-1)
        y = np.where(fine[..., None], y, np.float32(0))
        lo = y.min(-1) + np.float32(0)
        s = _FP16[np.searchsorted(15.0 * _FP16, (y.max(-1) - lo).astype(np.float64))]
        n = np.where(s[..., None] > 0, np.rint((y - lo[..., None]).astype(np.float64) / np.where(s > 0, s, 1.0)[..., None]), 0.0)
    lo = np.where(fine, lo, np.nan).astype(np.float16)
    return n.astype(np.int64), lo, np.where(fine, s, 0.0).astype(np.float16)


def values(n: np.ndarray, lo: np.ndarray, s: np.ndarray) -> np.ndarray:
    return lo.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * n


def key_place(slot: int, dim: int) -> Tuple[int, int]:
    """(byte of the unit, lowest bit in it) of a K level."""
    i, e = divmod(slot, 4)
    x, rest = divmod(dim, 32)
    g, j = divmod(rest, 8)
    bit = 4 * (j // 2) + 16 * (j % 2)
    return 256 * (i // 2) + 64 * e + 16 * g + 8 * (i % 2) + 4 * x + bit // 8, bit % 8


def value_place(slot: int, dim: int) -> Tuple[int, int]:
    q, t = divmod(slot, 4)
    p, rest = divmod(dim, 32)
    high, r = divmod(rest, 16)
    return 512 + 256 * (q // 2) + 16 * r + 8 * (q % 2) + 4 * p + (0, 2, 1, 3)[t], 4 * high


def pair_place(kind: int, slot: int) -> int:
    return 1024 + 64 * kind + 4 * slot


_PLACES = np.array([[[place(t, d) for d in range(DIM)] for t in range(SLOTS)] for place in (key_place, value_place)])


def write(pool: np.ndarray, layer_begin: int, key: np.ndarray, value: np.ndarray, slots: Sequence[int]) -> None:
    """The append into pool uint8 [22, blocks, 4, 1152] (in place): key/value float16 [layers, tokens, 4, 64]; slots outside
    the pool are skipped."""
    for kind, rows in enumerate((key, value)):
        n, lo, s = quantize(rows)
        for token, slot in enumerate(slots):
            if not 0 <= slot < pool.shape[1] * SLOTS:
                continue
            block, t = divmod(int(slot), SLOTS)
            units = pool[layer_begin : layer_begin + key.shape[0], block]  # [layers, 4, 1152]
            for d in range(DIM):
                byte, bit = _PLACES[kind, t, d]
                units[..., byte] = units[..., byte] & ~np.uint8(15 << bit) | (n[:, token, :, d] << bit).astype(np.uint8)
            at = pair_place(kind, t)
            units[..., at : at + 4] = np.stack((lo[:, token], s[:, token]), axis=-1).view(np.uint8)


def rows(units: np.ndarray, kind: int, slots: np.ndarray) -> np.ndarray:
    """The values in 64 bits, [tokens, 4, 64], of the rows at `slots` of one layer, uint8 [blocks, 4, 1152]."""
    block, t = np.divmod(np.asarray(slots), SLOTS)
    places = _PLACES[kind][t]  # [tokens, 64, 2]
    taken = units[block]  # [tokens, 4, 1152]
    n = np.take_along_axis(taken, np.broadcast_to(places[:, None, :, 0], (len(t), HEADS, DIM)), axis=-1) >> places[:, None, :, 1] & 15
    at = (1024 + 64 * kind + 4 * t)[:, None, None] + np.arange(4)
    pair = np.take_along_axis(taken, np.broadcast_to(at, (len(t), HEADS, 4)), axis=-1).copy().view(np.float16)
    return values(n.astype(np.int64), pair[..., 0], pair[..., 1])


def attention(query: np.ndarray, units: np.ndarray, table: Sequence[int], length: int) -> Tuple[np.ndarray, np.ndarray]:
    """softmax(q . K^T / 8) V in 64 bits for query float16 [32, 64], and how far an fp32 evaluation with one rounding to
    fp16 may be from it, both [32, 64].

    The bound, to first order and doubled: a score is 64 products and a few roundings of 2^-24 of its terms' magnitudes, so
    each weight is off by that over 8, by the exponential's own 2^-21 and by the rounding of its argument; the weights that
    multiply the levels keep 16 bits; sums run over length / 32 (matrix instruction, levels up to 15 beside an offset of
    128) or length / 8 (a lane's) additions and 80 at the joins."""
    slots = np.array([table[p // SLOTS] * SLOTS + p % SLOTS for p in range(length)])
    k, v = rows(units, 0, slots), rows(units, 1, slots)
    q = query.astype(np.float64)
    out, bound = np.empty((32, DIM)), np.empty((32, DIM))
    for head in range(32):
        kh, vh = k[:, head // 8], v[:, head // 8]
        y = kh @ q[head] / 8.0
        p = np.exp(y - y.max())
        p /= p.sum()
        out[head] = p @ vh
        low = vh.min()
        span, size = np.abs(vh.max(0) - low).max(), np.abs(vh).max()
        lo_k = np.abs(kh).max(1) + (kh.max(1) - kh.min(1))  # >= |lo| and >= 15 s
        score = 80 * 2.0**-24 * 2 * np.abs(q[head]).sum() * lo_k.max() / 8.0
        weight = score + 2.0**-21 + 2.0**-22 * min(np.abs(y - y.max()).max(), 20.0)
        row_span = (vh.max(1) - vh.min(1)).max()
        add = (length / 32 + 80) * 2.0**-24 * (143.0 / 15.0) * row_span + (length / 8 + 80) * 2.0**-24 * size
        spread = min(2 * size, span)
        bound[head] = 2.0**-11 * np.abs(out[head]) + 2.0**-25 + 2 * (weight * spread + 2.0**-17 * row_span + add + (length / 8 + 80) * 2.0**-24 * np.abs(out[head]))
    return out, bound
