"""The bound that attention over the 4-bit pool is held to tells a right evaluation from wrong ones (CPU only)."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import q4_reference as ref
from tests.q4_cases import CASES, build


def _evaluate(query, units, table, length, *, scale=1.0, weight_bits=16, wrong_half=False, whole_group=False):
    """attention() in fp32, or with a mistake: the softmax's scale off, weights of fewer bits, a large query's sixteenths at the wrong
    places, or rounded to fp16 for all heads of a group where one of them is large."""
    slots = np.array([table[p // 16] * 16 + p % 16 for p in range(length)])
    out = np.empty((32, 64), dtype=np.float16)
    k, v = (ref.rows(units, kind, slots) for kind in range(2))
    for head in range(32):
        q = query[head].astype(np.float32)
        kh, vh = k[:, head // 8].astype(np.float32), v[:, head // 8]
        if wrong_half and (np.abs(q) >= 4096).any():
            q = np.where(np.isin(np.arange(64) % 8, (0, 1, 4, 5)), q / 16, q * 16).astype(np.float32)
        if whole_group and (np.abs(query[head // 8 * 8 : head // 8 * 8 + 8].astype(np.float32)) >= 4096).any():
            q = np.where(np.isin(np.arange(64) % 8, (2, 3, 6, 7)), (q / 16).astype(np.float16).astype(np.float32) * 16, q)
        y = kh @ q
        p = np.exp((y - y.max()) * np.float32(scale / 8.0)).astype(np.float64)
        low = vh.min(1, keepdims=True)
        weights = p.copy()
        if weight_bits < 16:
            mantissa, exponent = np.frexp(weights)
            weights = np.ldexp(np.round(mantissa * 2.0**weight_bits) / 2.0**weight_bits, exponent)
        out[head] = ((weights @ (vh - low) + p @ low) / p.sum()).astype(np.float16)
    return out


def _share(case, **wrong):
    query, pool, tables, lengths = build(case)
    worst = 0.0
    for b, length in enumerate(lengths):
        want, bound = ref.close_attention(query[b], pool, tables[b], length)
        loose, _ = ref.attention(query[b], pool, tables[b], length)
        assert np.allclose(want, loose, rtol=1e-12, atol=1e-12)
        got = np.zeros((32, 64)) if wrong.get("zeros") else _evaluate(query[b], pool, tables[b], length, **wrong).astype(np.float64)
        worst = max(worst, float((np.abs(got - want) / bound).max()))
    return worst


@pytest.mark.parametrize("case", list(CASES))
def test_a_right_evaluation_is_within(case):
    assert _share(case) <= 1.0


@pytest.mark.parametrize("case", list(CASES))
def test_zeros_are_not(case):
    assert _share(case, zeros=True) > 4.0


@pytest.mark.parametrize("case", ["short", "ordinary", "rising"])
def test_a_softmax_of_another_scale_is_not(case):
    assert _share(case, scale=1.01) > 1.5


@pytest.mark.parametrize("case", ["short", "ordinary"])
def test_weights_of_one_bf16_are_not(case):
    assert _share(case, weight_bits=8) > 1.5


@pytest.mark.parametrize("case", ["large elements", "one large element"])
def test_sixteenths_at_the_wrong_places_are_not(case):
    assert _share(case, wrong_half=True) > 4.0


def test_sixteenths_of_small_heads_beside_a_large_one_are_not():
    assert _share("large and small heads", whole_group=True) > 4.0
    assert _share("one large element", whole_group=True) <= 1.0  # 16 bits of ordinary elements stay
