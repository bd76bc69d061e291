"""Decode steps of a serving batch over a 4-bit KV pool: more rows than eight, contexts of several hundred tokens, so that the
graph's attention takes two waves a kv head over bins of several sequences and over cut ones, behind a padded plan."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import q4_reference as ref
from pagedcore_amd import decoder as dec
from pagedcore_amd.engine_types import KVReservation, RequestId
from pagedcore_amd.kv_cache import KVAllocator

pytestmark = pytest.mark.gpu

LENGTHS = [1, 40, 700, 16, 333, 1500, 64, 900, 129, 17, 2000, 250]


def _allocator(device):
    pool = torch.zeros((22, 420, 4, 1152), dtype=torch.uint8, device=device)
    return KVAllocator(pool)


def _fill(allocator, device):
    """Requests whose cached rows are random, the same in each allocator."""
    gen = torch.Generator(device=device).manual_seed(4)
    requests = []
    for i, length in enumerate(LENGTHS):
        request = RequestId(f"r{i}")
        allocator.create(KVReservation(request, -(-(length + 8) // 16)))
        key, value = (torch.randn(22, length, 4, 64, dtype=torch.float16, device=device, generator=gen) for _ in range(2))
        allocator.append(request, key, value)
        requests.append(request)
    return requests


@pytest.mark.parametrize("rows", [12, 16])
def test_steps(device, rows, monkeypatch):
    small = dec.random_weights(device=device, seed=11, layers=2, vocab=31, intermediate=32, norm_std=0.1)
    weights = dec.TinyLlamaWeights(small.embedding, small.layers * 11, small.final_norm, small.lm_head)
    eager, captured = _allocator(device), _allocator(device)
    requests = _fill(eager, device)
    assert _fill(captured, device) == requests and torch.equal(eager.pool, captured.pool)
    attended = []
    original = dec.attend_rows

    def attend(query, allocator, request_ids, layer):
        out, workspace = original(query, allocator, request_ids, layer)
        if layer == 13:
            attended.append((query.cpu().numpy(), out.cpu().numpy(), allocator.pool[layer].cpu().numpy()))
        return out, workspace

    monkeypatch.setattr(dec, "attend_rows", attend)
    graph = dec.DecodeGraph(weights, captured, rows)
    for step in range(3):
        order = tuple(requests if step != 1 else reversed(requests))
        tokens = torch.tensor([[(5 * step + i) % 31] for i in range(12)], device=device)
        expected = dec.decode_paged(tokens, weights, eager, order)
        got = graph.step(tokens, order)
        graph.check_faults()
        if rows == 12:  # of more rows the projections may add in another order
            assert torch.equal(got.view(torch.int16), expected.view(torch.int16))
            assert torch.equal(eager.pool, captured.pool)
        else:
            assert torch.isfinite(got).all()
    for query, out, units in attended[:1]:
        for b, (request, length) in enumerate(zip(requests, LENGTHS)):
            want, bound = ref.close_attention(query[b, :, 0], units, eager.block_table(request), length + 1)
            assert (np.abs(out[b, :, 0].astype(np.float64) - want) <= bound).all(), request
