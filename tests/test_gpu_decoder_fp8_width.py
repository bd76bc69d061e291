"""The 8-bit model at the MLP width of TinyLlama (5632), where its projections take the kernels that they take in use:
SwiGLU of a decode step's rows the tiles too, long prompts the wide ones (tests/test_gpu_decoder_fp8.py has narrow MLPs)."""

from __future__ import annotations

import pytest
import torch

from oracle import decoder_reference as dref
from pagedcore_amd import decoder as dec
from pagedcore_amd.engine_types import KVReservation, RequestId
from pagedcore_amd.kv_cache import KVAllocator
from tests.test_gpu_decoder_fp8 import _allocator, _host, _no_further, _oracle, _admit, _weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights():
    return _weights(torch.device("cuda:0"), intermediate=dec.INTERMEDIATE)[1]


def _pools(device, blocks):
    return [torch.full((22, 2, blocks, 16, 4, 64), float("nan"), dtype=torch.float16, device=device) for _ in range(2)]


@pytest.mark.parametrize("batch", [1, 24, 40, 100, 150, 200])
def test_decode_graph_equals_decode_paged(device, weights, batch):
    pools = _pools(device, 2 * batch)
    eager, graphed = (KVAllocator(pool) for pool in pools)
    requests = tuple(RequestId(f"g{row}") for row in range(batch))
    for row, request in enumerate(requests):
        ids = ((torch.arange(1 + row % 18)[None] * 3 + row) % 31).to(device)
        for allocator in (eager, graphed):
            allocator.create(KVReservation(request, 2))
            dec.prefill_paged(ids, weights, allocator, request)
    graph = dec.DecodeGraph(weights, graphed, batch=batch)
    for step in range(3):
        tokens = torch.tensor([[(5 * step + row) % 31] for row in range(batch)], device=device)
        expected = dec.decode_paged(tokens, weights, eager, requests)
        assert torch.equal(graph.step(tokens, requests), expected)
        graph.check_faults()
        assert torch.equal(pools[0].view(torch.int16), pools[1].view(torch.int16))


@pytest.mark.parametrize("tokens", [24, 150, 333, 700, 1100, 2040])
def test_prefill_graph_writes_the_cache_of_prefill_paged(device, weights, tokens):
    pools = _pools(device, 130)
    eager, graphed = (KVAllocator(pool) for pool in pools)
    graph = dec.PrefillGraph(weights, graphed, tokens)
    request = RequestId("p")
    for turn in range(2):
        ids = ((torch.arange(tokens) * 3 + turn) % 31)[None].to(device)
        for allocator in (eager, graphed):
            allocator.create(KVReservation(request, (tokens + 15) // 16))
        expected = dec.prefill_paged(ids, weights, eager, request)
        got = graph.step(ids, request)
        assert torch.equal(pools[0].view(torch.int16), pools[1].view(torch.int16))
        torch.testing.assert_close(got[0, 0], expected[0, -1], atol=5e-3, rtol=5e-3)  # the LM head at another row count
        for allocator in (eager, graphed):
            allocator.release_all(request)


def test_prefill_is_as_close_as_the_oracle(device, weights):
    host = _host(weights)
    ids = (torch.arange(333) * 7 + 5) % 31
    _, logits = _admit(_allocator(device), weights, "p", ids[None].to(device))
    exact, _ = dref.forward(ids[None], host, fp32_attention=True)
    _no_further(logits[0].float(), _oracle(ids, host), exact[0])
