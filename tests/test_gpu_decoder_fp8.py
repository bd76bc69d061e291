"""The decoder on 8-bit projections: quantize_weights, and prefill, decode, their graphs and the worker on its result.

The rounding of an activation to e4m3 may fall to either side where two computations differ in their
last bits, and moves a value by up to 2^-4: logits are not compared element by element. The
measure is the distance (2-norm) from the same 8-bit weights applied without rounding activations, in
fp32: the GPU's may be at most 1.25 times that of the oracle's evaluation, which rounds where the
kernels round. What is computed twice by the same kernels is compared bit for bit.
"""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import decoder_reference as dref
from oracle import fp8_reference as ref
from pagedcore_amd import _hip
from pagedcore_amd import decoder as dec
from pagedcore_amd.engine_types import KVReservation, RequestId
from pagedcore_amd.kv_cache import KVAllocator
from pagedcore_amd.worker import DecodeWorker, FinishReason, GenerationRequest

pytestmark = pytest.mark.gpu

Q, KV = 2048, 256


def _weights(device, intermediate=32, vocab=31, seed=11):
    """Two distinct layers repeated 11 times, fp16 and in 8 bits (repeated likewise)."""
    small = dec.random_weights(device=device, seed=seed, layers=2, vocab=vocab, intermediate=intermediate, norm_std=0.1)
    eight = dec.quantize_weights(small)
    many = lambda w: dec.TinyLlamaWeights(w.embedding, w.layers * 11, w.final_norm, w.lm_head)  # noqa: E731
    return many(small), many(eight)


def _stands(rows: dec.Fp8Rows) -> torch.Tensor:
    return ref.stands_for(rows.values.cpu(), rows.scales.cpu().view(torch.uint8).long()).float()


def _host(weights):
    """The 8-bit weights' values in fp32 on the CPU, under the oracle's field names."""
    built = {}
    for layer in weights.layers:
        if id(layer) not in built:
            qkv, gate_up = _stands(layer.qkv), _stands(layer.gate_up)
            half = gate_up.shape[0] // 2
            built[id(layer)] = SimpleNamespace(
                input_norm=layer.input_norm.cpu().float(), q_proj=qkv[:Q], k_proj=qkv[Q : Q + KV], v_proj=qkv[Q + KV :],
                o_proj=_stands(layer.o_proj), post_attention_norm=layer.post_attention_norm.cpu().float(), gate_proj=gate_up[:half],
                up_proj=gate_up[half:], down_proj=_stands(layer.down_proj), qkv=qkv,
            )
    return SimpleNamespace(
        embedding=weights.embedding.cpu().float(), layers=tuple(built[id(layer)] for layer in weights.layers),
        final_norm=weights.final_norm.cpu().float(), lm_head=weights.lm_head.cpu().float(),
    )


def _round(x: torch.Tensor) -> torch.Tensor:
    """What rows rounded to 8 bits stand for, in fp32."""
    values, s = ref.round_rows(x.double())
    return ref.stands_for(values, s).float()


def _oracle(ids: torch.Tensor, host) -> torch.Tensor:
    """Logits [tokens, vocab] of the contiguous forward, rounding where the kernels round: the residual and
    each projection's output to fp16, each projection's input to 8 bits."""
    norm = lambda h, w: (h.double() / torch.sqrt(h.double().square().mean(-1, keepdim=True) + 1e-5) * w.double()).float()  # noqa: E731
    tokens = ids.numel()
    positions = torch.arange(tokens)[None]
    allowed = torch.ones((tokens, tokens), dtype=torch.bool).tril()[None, None]
    hidden = host.embedding[ids]
    for layer in host.layers:
        qkv = (_round(norm(hidden, layer.input_norm)) @ layer.qkv.t()).half()
        heads = qkv.view(1, tokens, 40, 64).transpose(1, 2)
        query, key = dref.apply_rope(heads[:, :32], heads[:, 32:36], positions)
        attention = dref.dense_attention_fp32(query, key, heads[:, 36:], allowed)[0].transpose(0, 1).reshape(tokens, Q)
        hidden = (hidden + (_round(attention.float()) @ layer.o_proj.t()).half().float()).half().float()
        x = _round(norm(hidden, layer.post_attention_norm))
        gate, up = x @ layer.gate_proj.t(), x @ layer.up_proj.t()
        active = gate / (1 + torch.exp(-gate)) * up
        hidden = (hidden + (_round(active) @ layer.down_proj.t()).half().float()).half().float()
    return norm(hidden, host.final_norm) @ host.lm_head.t()


def _no_further(got, oracle, exact):
    distance = lambda a: (a.cpu().double() - exact.double()).norm().item()  # noqa: E731
    assert distance(got) <= 1.25 * distance(oracle), (distance(got), distance(oracle))


def _allocator(device, blocks=64):
    return KVAllocator(torch.full((22, 2, blocks, 16, 4, 64), float("nan"), dtype=torch.float16, device=device))


def _admit(allocator, weights, name, ids, spare=16):
    request = RequestId(name)
    allocator.create(KVReservation(request, (ids.shape[1] + spare + 15) // 16))
    return request, dec.prefill_paged(ids, weights, allocator, request)


def test_quantize_weights_rounds_every_projection(device):
    half, eight = _weights(device, intermediate=48)
    for layer, rounded in zip(half.layers[:2], eight.layers[:2]):
        for rows, parts in ((rounded.qkv, (layer.q_proj, layer.k_proj, layer.v_proj)), (rounded.o_proj, (layer.o_proj,)),
                            (rounded.gate_up, (layer.gate_proj, layer.up_proj)), (rounded.down_proj, (layer.down_proj,))):
            values, s = ref.round_rows(torch.cat(parts).cpu().double())
            assert torch.equal(rows.values.cpu().double(), values)
            assert torch.equal(rows.scales.cpu().view(torch.uint8)[:, : s.shape[1]].long(), s)
        assert rounded.input_norm is layer.input_norm and rounded.post_attention_norm is layer.post_attention_norm
    assert eight.embedding is half.embedding and eight.lm_head is half.lm_head


def test_quantize_weights_refuses(device):
    half, eight = _weights(device)
    with pytest.raises(ValueError, match="already in 8 bits"):
        dec.quantize_weights(eight)
    odd = dec.random_weights(device=device, layers=1, vocab=8, intermediate=24)
    with pytest.raises(ValueError, match="multiple of 16"):
        dec.quantize_weights(odd)
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        dec.quantize_weights(dec.random_weights(device="cpu", layers=1, vocab=8, intermediate=16))


@pytest.mark.parametrize("tokens", [1, 17, 49, 140])
def test_prefill_is_as_close_as_the_oracle(device, tokens):
    _, weights = _weights(device, intermediate=272)
    host = _host(weights)
    ids = (torch.arange(tokens) * 7 + tokens) % 31
    _, logits = _admit(_allocator(device), weights, "p", ids[None].to(device))
    exact, _ = dref.forward(ids[None], host, fp32_attention=True)
    _no_further(logits[0].float(), _oracle(ids, host), exact[0])


@pytest.mark.parametrize("batch", [1, 5, 40])
def test_decode_is_as_close_as_the_oracle(device, batch):
    """Every row's next-token logits, against the contiguous forward of its prompt and new token."""
    _, weights = _weights(device, intermediate=272)
    host = _host(weights)
    allocator = _allocator(device, 40 * 4)
    requests, prompts = [], []
    for row in range(batch):
        ids = (torch.arange(3 + row % 20) * 5 + row) % 31
        requests.append(_admit(allocator, weights, f"r{row}", ids[None].to(device))[0])
        prompts.append(ids)
    new = torch.tensor([[(3 * row + 1) % 31] for row in range(batch)], device=device)
    logits = dec.decode_paged(new, weights, allocator, tuple(requests))
    oracle, exact = [], []
    for row in range(0, batch, 4):
        ids = torch.cat((prompts[row], new[row].cpu()))
        oracle.append(_oracle(ids, host)[-1])
        exact.append(dref.forward(ids[None], host, fp32_attention=True)[0][0, -1])
    _no_further(logits[::4, 0].float(), torch.stack(oracle), torch.stack(exact))


@pytest.mark.parametrize("batch", [1, 7, 33, 65, 130])
def test_decode_graph_replays_equal_decode_paged(device, batch):
    """One captured step replayed with eager work between: logits and cache bytes of decode_paged, bit for bit, at
    row counts of every route of the projections."""
    _, weights = _weights(device, intermediate=176)
    pools = [torch.full((22, 2, batch * 3 + 4, 16, 4, 64), float("nan"), dtype=torch.float16, device=device) for _ in range(2)]
    eager, graphed = (KVAllocator(pool) for pool in pools)
    requests = tuple(RequestId(f"g{row}") for row in range(batch))
    for row, request in enumerate(requests):
        ids = ((torch.arange(1 + row % 18)[None] * 3 + row) % 31).to(device)
        for allocator in (eager, graphed):
            allocator.create(KVReservation(request, 3))
            dec.prefill_paged(ids, weights, allocator, request)
    graph = dec.DecodeGraph(weights, graphed, batch=batch)
    for step in range(4):
        order = requests if step % 2 == 0 else tuple(reversed(requests))
        tokens = torch.tensor([[(5 * step + row) % 31] for row in range(batch)], device=device)
        expected = dec.decode_paged(tokens, weights, eager, order)
        got = graph.step(tokens, order)
        graph.check_faults()
        assert torch.equal(got, expected)
        assert torch.equal(pools[0].view(torch.int16), pools[1].view(torch.int16))
        torch.randn(1000, device=device).sum().item()  # unrelated eager work between replays


@pytest.mark.parametrize("tokens", [16, 50, 200])
def test_prefill_graph_equals_prefill_paged(device, tokens):
    """Cache bytes of prefill_paged at the graph's own size; a shorter prompt pads and stays as close as the oracle."""
    _, weights = _weights(device, intermediate=176)
    host = _host(weights)
    pools = [torch.full((22, 2, 40, 16, 4, 64), float("nan"), dtype=torch.float16, device=device) for _ in range(2)]
    eager, graphed = (KVAllocator(pool) for pool in pools)
    graph = dec.PrefillGraph(weights, graphed, tokens)
    for turn in range(3):
        ids = ((torch.arange(tokens) * 3 + turn) % 31)[None].to(device)
        request, expected = _admit(eager, weights, f"t{turn}", ids)
        graphed.create(KVReservation(request, (tokens + 31) // 16))
        got = graph.step(ids, request)
        assert torch.equal(pools[0].view(torch.int16), pools[1].view(torch.int16))
        torch.testing.assert_close(got[0, 0], expected[0, -1], atol=5e-3, rtol=5e-3)  # the LM head at another row count
        for allocator in (eager, graphed):
            allocator.release_all(request)
    short = (torch.arange(tokens - 3) * 5) % 31
    request = RequestId("short")
    graphed.create(KVReservation(request, (tokens + 15) // 16))
    got = graph.step(short[None].to(device), request)
    exact, _ = dref.forward(short[None], host, fp32_attention=True)
    _no_further(got[0].float(), _oracle(short, host)[-1:], exact[0, -1:])


def test_worker_serves_8_bit_weights(device):
    """Requests through captured graphs and eagerly: every one finishes, and one alone matches a loop by hand."""
    _, weights = _weights(device, intermediate=176)
    for graphs in ({}, {"graph_batch": (2, 4), "prefill_graph_tokens": (16,)}):
        worker = DecodeWorker(weights, _allocator(device), max_active=4, **graphs)
        for i in range(6):
            worker.submit(GenerationRequest(RequestId(f"w{i}"), tuple((3 * i + j) % 31 for j in range(4 + 3 * i)), 5, ignore_eos=True))
        results = worker.run(max_steps=60)
        assert len(results) == 6 and all(len(r.greedy_ids) == 5 and r.finish_reason is FinishReason.LENGTH for r in results.values())
    worker = DecodeWorker(weights, _allocator(device), max_active=1)
    worker.submit(GenerationRequest(RequestId("one"), (1, 5, 9), 4, ignore_eos=True))
    alone = worker.run(max_steps=20)[RequestId("one")].greedy_ids
    allocator = _allocator(device)
    request, logits = _admit(allocator, weights, "one", torch.tensor([[1, 5, 9]], device=device))
    chosen = [int(logits[0, -1].argmax())]
    for _ in range(3):
        chosen.append(int(dec.decode_paged(torch.tensor([[chosen[-1]]], device=device), weights, allocator, (request,))[0, -1].argmax()))
    assert tuple(chosen) == alone


def test_the_chain_of_a_layer_equals_its_operators(device):
    """norm, SwiGLU, down projection and norm, as the decoder runs them on a side stream, against the same
    operators one at a time on the default stream with synchronizations between."""
    _, weights = _weights(device, intermediate=176)
    layer = weights.layers[0]
    hidden = torch.randn(24, 2048, device=device).half()
    outputs = []
    for wait in (False, True):
        stream = torch.cuda.current_stream() if wait else torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            h = hidden.clone()
            x = dec._norm_fp8(h, None, layer.input_norm)
            pause = torch.cuda.synchronize if wait else (lambda: None)
            pause()
            active = torch.empty((24, 176), dtype=torch.float16, device=device)
            _hip.gemm_fp8(active, x.values, x.scales, layer.gate_up.values, layer.gate_up.scales, epilogue=_hip.GEMM_SWIGLU)
            pause()
            parts = torch.empty((2, 24, 2048), device=device)
            _hip.gemm_fp8(parts, active, None, layer.down_proj.values, layer.down_proj.scales, splits=2)
            pause()
            y = dec._norm_fp8(h, parts, layer.post_attention_norm)
        torch.cuda.synchronize()
        outputs.append((h, y.values.view(torch.uint8), y.scales.view(torch.uint8)))
    for a, b in zip(*outputs):
        assert torch.equal(a, b)
