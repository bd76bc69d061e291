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
    multiply the levels keep 16 bits; sums run over length / 32 (matrix instruction, levels up to 15 beside an offset, for
    which 128 is allowed) or length / 8 (a lane's) additions and 80 at the joins."""
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


def close_attention(query: np.ndarray, units: np.ndarray, table: Sequence[int], length: int) -> Tuple[np.ndarray, np.ndarray]:
    """attention() with a bound that goes by each token's own error and weight, [32, 64].

    With u = 2^-24 and the formula y = s (q . n) + lo sum(q), before the division by 8: the two sums are 64 exact products each,
    added in any order (64 u of their terms' magnitudes); the running maximum m, at most the largest |y|, is taken off within
    the second product and again wherever it is raised (by 8 binary orders or more) or two parts meet. A head with an element of
    thousands (squares of its sixteenths past 65500) has half of its elements divided by 16, to within 2^-21 of an element. These
    make token t's exponent off by e_t, and with the roundings of the base-2 exponential and its argument its weight by
    d_t = exp(e_t + ...) - 1, which moves the output by p_t d_t |v_t - out|, and by no more than the values spread. Weights
    times steps keep 17 bits of the levels' product; levels enter it as 16 + n, and n / 32 products and 56 joins are rounded, of the
    minima's and the weights' sums length / 8 and 16 additions a lane. Then the rounding to fp16."""
    u = 2.0**-24
    slots = np.array([table[p // SLOTS] * SLOTS + p % SLOTS for p in range(length)])
    block, t = np.divmod(slots, SLOTS)
    out, bound = np.empty((32, DIM)), np.empty((32, DIM))
    q = query.astype(np.float64)
    halved = np.isin(np.arange(DIM) % 8, (2, 3, 6, 7))
    for kv in range(HEADS):
        fields = []
        for kind in range(2):
            taken = units[block, kv]  # [tokens, 1152]
            places = _PLACES[kind][t]
            n = np.take_along_axis(taken, places[..., 0], axis=-1) >> places[..., 1] & 15
            pair = np.take_along_axis(taken, (1024 + 64 * kind + 4 * t)[:, None] + np.arange(4), axis=-1).copy().view(np.float16).astype(np.float64)
            fields.append((n.astype(np.float64), pair[:, :1], pair[:, 1:]))
        (kn, klo, ks), (vn, vlo, vs) = fields
        v = vlo + vs * vn
        for head in range(8 * kv, 8 * kv + 8):
            size = np.abs(q[head]).sum()
            y = (klo + ks * kn) @ q[head]
            most = np.abs(y).max()
            span = (y.max() - y.min()) / 8.0
            raises = 1 + min(span / np.log(2.0) / 8.0, length / 64)
            error = 64 * u * (ks[:, 0] * (kn @ np.abs(q[head])) + np.abs(klo[:, 0]) * size) + u * (np.abs(klo[:, 0] * q[head].sum()) + (4 + 2 * raises + 8) * most)
            if ((q[head] / 16) ** 2).sum() > 65400:
                error = error + 2.0**-21 * ks[:, 0] * kn[:, halved].sum(1)
            z = (y - y.max()) / 8.0
            p = np.exp(z)
            p /= p.sum()
            with np.errstate(over="ignore"):
                d = np.expm1(error / 8.0 + 3 * u * np.minimum(-z, 100.0) + (3 + raises) * 2.0**-22 + 16 * 2.0**-23)
            out[head] = p @ v
            apart = np.abs(v - out[head])
            moved = np.minimum((p * np.minimum(d, 1e300)) @ apart, np.abs(v.max(0) - v.min(0)))
            steps = p @ vs
            levels = (p[:, None] * vs * (16 + vn)).sum(0) + 16 * steps
            lane = length / 8 + 16
            bound[head] = (
                2.0**-11 * np.abs(out[head]) + 2.0**-25 + 1.01 * moved + 2.0**-17 * (p[:, None] * vs * vn).sum(0)
                + u * ((length / 32 + 56) * levels + lane * (p @ np.abs(vlo)) + lane * np.abs(out[head]))
            )
    return out, bound
