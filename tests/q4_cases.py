"""Queries and 4-bit pools of a layer whose attention is well conditioned, so that it can be held to a bound near fp16's rounding."""

from __future__ import annotations

import numpy as np

from oracle import q4_reference as ref


def _ordinary(rng, lengths, tokens):
    query = rng.standard_normal((len(lengths), 32, 64)).astype(np.float16)
    key, value = (rng.standard_normal((1, tokens, 4, 64)).astype(np.float16) for _ in range(2))
    return query, key, value


def _on_levels(rng, tokens, step, zero_dims=()):
    """Key rows step (n - 8), both ends among the levels, 0 in `zero_dims`."""
    n = rng.integers(0, 16, (1, tokens, 4, 64))
    n[..., 62], n[..., 63] = 0, 15
    n[..., list(zero_dims)] = 8
    return (step * (n - 8.0)).astype(np.float16)


def _large(elements):
    """Queries of ordinary size but for given elements ({dim: value}), which meet keys of 0 there and so change no score."""

    def make(rng, lengths, tokens):
        query, _, value = _ordinary(rng, lengths, tokens)
        key = _on_levels(rng, tokens, 2.0**-6, [d for d in elements if d < 62])
        for dim, values in elements.items():
            query[:, ::2, dim] = np.resize(np.array(values, dtype=np.float16), 16)
        return query, key, value

    return make


def _large_and_small_heads(rng, lengths, tokens):
    """Head 0 of each group has an element of 4096 to 65504; the others' are of 2^-15, over keys to 32768."""
    query, _, value = _ordinary(rng, lengths, tokens)
    query = (query.astype(np.float64) * 2.0**-15).astype(np.float16)
    query[:, 0::8, 10] = np.array([4096, 65504, -65504, 8192], dtype=np.float16)
    return query, _on_levels(rng, tokens, 4096.0, [10]), value


def _one_wins(rng, lengths, tokens):
    """Queries to 60000 in every element along one token's key: its value, and no other's, is what comes out."""
    key = _on_levels(rng, tokens, 2.0**-3)
    value = rng.standard_normal((1, tokens, 4, 64)).astype(np.float16)
    return None, key, value


def _rising(rng, lengths, tokens):
    """Scores that rise along a sequence, by 14 binary orders a step of 64 tokens: the running maximum is raised at every step."""
    query, key, value = _ordinary(rng, lengths, tokens)
    return query, key, value


CASES = {
    "short": (_ordinary, [1, 2, 5, 16, 17, 40]),
    "ordinary": (_ordinary, [130, 700]),
    "large elements": (_large({d: [4094, 4096, 65504, -65504, 5000, -4098] for d in (0, 2, 13, 31, 32, 38, 55, 61)}), [90, 33]),
    "one large element": (_large({3: [65504, -65504]}), [64, 200]),
    "border": (_large({4: [4094, -4094], 6: [4092]}), [64, 200]),
    "large and small heads": (_large_and_small_heads, [50, 300]),
    "one wins": (_one_wins, [70, 260]),
    "rising": (_rising, [512, 300]),
}


def build(name, lengths=None, seed=0):
    """(query float16 [batch, 32, 64], units uint8 [blocks, 4, 1152], tables, lengths) of a case."""
    make, own_lengths = CASES[name]
    lengths = own_lengths if lengths is None else lengths
    rng = np.random.default_rng(seed + len(name))
    need = [-(-n // 16) for n in lengths]
    ids = rng.permutation(sum(need))
    tables = np.zeros((len(lengths), max(need)), dtype=np.int32)
    for b, n in enumerate(need):
        tables[b, :n] = ids[sum(need[:b]) : sum(need[: b + 1])]
    tokens = 16 * len(ids)
    query, key, value = make(rng, lengths, tokens)
    slots = [np.array([tables[b, p // 16] * 16 + p % 16 for p in range(n)]) for b, n in enumerate(lengths)]
    if name == "one wins":
        query = np.empty((len(lengths), 32, 64), dtype=np.float16)
        for b, n in enumerate(lengths):
            winner = key[0, slots[b][n // 3]].astype(np.float64)  # [4, 64]
            scale = np.resize([60000.0, 30000.0, 4096.0, 512.0], 8)[None, :, None]
            query[b] = (winner[:, None, :] * scale).reshape(32, 64).astype(np.float16)
    if name == "rising":
        # A third of every key along the first query of its group's sum, ever longer.
        for b, n in enumerate(lengths):
            query[b] = np.repeat(query[b, ::8], 8, axis=0) + 0.25 * query[b]
            along = query[b, ::8].astype(np.float64)
            rise = 14 * np.log(2.0) / 64 * np.arange(n) * 8.0 / (along**2).sum(-1)[:, None]  # [4, tokens]
            rows = 0.3 * key[0, slots[b]].astype(np.float64) + (rise[..., None] * along[:, None]).transpose(1, 0, 2)
            key[0, slots[b]] = rows.astype(np.float16)
    units = rng.integers(0, 256, (22, len(ids), 4, ref.UNIT), dtype=np.uint8)
    ref.write(units, 0, key, value, range(tokens))
    return query, units[0], tables, list(lengths)
