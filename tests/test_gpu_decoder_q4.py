"""The allocator, the decoder, its graphs and the worker over a 4-bit KV pool.

What two paths compute with the same kernels is compared bit for bit: a prompt's logits with the fp16 pool's, its cache with
the fp16 pool's rows quantised, a DecodeGraph with decode_paged, the worker's tokens with requests generated alone."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import q4_reference as ref
from pagedcore_amd import _hip
from pagedcore_amd import decoder as dec
from pagedcore_amd.attention import paged_attention, paged_attention_batch
from pagedcore_amd.config import PagedCoreConfig
from pagedcore_amd.engine_types import KVReservation, RequestId
from pagedcore_amd.kv_cache import HipQ4Writer, KVAllocator, allocate_kv_pool
from pagedcore_amd.worker import DecodeWorker, GenerationRequest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights():
    small = dec.random_weights(device="cuda:0", seed=11, layers=2, vocab=31, intermediate=32, norm_std=0.1)
    return dec.TinyLlamaWeights(small.embedding, small.layers * 11, small.final_norm, small.lm_head)


def _q4(device, blocks=40, seed=0):
    """An allocator over a 4-bit pool of random bytes (NaN and infinities among them)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    return KVAllocator(torch.randint(0, 256, (22, blocks, 4, 1152), dtype=torch.uint8, device=device, generator=gen))


def _fp16(device, blocks=40):
    return KVAllocator(torch.full((22, 2, blocks, 16, 4, 64), float("nan"), dtype=torch.float16, device=device))


def _ids(device, length, seed):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, 31, (1, length))).to(device)


def _admit(allocator, weights, name, ids, spare=20):
    request = RequestId(name)
    allocator.create(KVReservation(request, -(-(ids.shape[1] + spare) // 16)))
    return request, dec.prefill_paged(ids, weights, allocator, request)


def _slots(allocator, request):
    table = np.asarray(allocator.block_table(request), dtype=np.int64)
    at = np.arange(allocator.cached_length(request))
    return table[at // 16] * 16 + at % 16


def _rows(allocator, request):
    """Every layer's K and V of the request, float16 [2, 22, tokens, 4, 64]."""
    slots = torch.from_numpy(_slots(allocator, request)).to(allocator.pool.device)
    out = torch.empty((2, 22, slots.shape[0], 4, 64), dtype=torch.float16, device=allocator.pool.device)
    _hip.kv_read_q4(out[0], out[1], allocator.pool, 0, slots)
    return out


@pytest.mark.parametrize("length", [1, 17, 130, 700, 1600])
def test_prefill(device, weights, length):
    ids = _ids(device, length, length)
    four, half = _q4(device, 120), _fp16(device, 120)
    before = four.pool.clone()
    request, logits = _admit(four, weights, "a", ids)
    other, expected = _admit(half, weights, "a", ids)
    assert torch.equal(logits.view(torch.int16), expected.view(torch.int16))
    assert four.block_table(request) == half.block_table(other) and four.cached_length(request) == length
    slots = torch.from_numpy(_slots(four, request)).to(device)
    rows = half.pool.view(22, 2, -1, 4, 64)[:, :, slots]
    _hip.kv_append_q4(before, 0, rows[:, 0].contiguous(), rows[:, 1].contiguous(), slots)
    assert torch.equal(four.pool, before)
    assert four.capacity() == half.capacity()


def test_allocator_writes_and_reads(device):
    allocator = _q4(device, 12)
    request = RequestId("a")
    allocator.create(KVReservation(request, 8))
    gen = torch.Generator(device=device).manual_seed(3)
    key, value = (torch.randn(22, 21, 4, 64, dtype=torch.float16, device=device, generator=gen) for _ in range(2))
    allocator.append(request, key[:, :20], value[:, :20])
    with allocator.append_decode((request,)):
        for layer in range(22):
            if layer % 2:
                allocator.write_decode_layer(request, layer, key[layer, 20], value[layer, 20])
            else:
                allocator.write_decode_layers((request,), layer, key[layer, 20:], value[layer, 20:])
    assert allocator.cached_length(request) == 21
    want = []
    for rows in (key, value):
        n, lo, step = ref.quantize(rows.cpu().numpy())
        want.append(ref.values(n, lo, step))
    for block, (begin, end) in enumerate(((0, 16), (16, 21))):
        for got, expected in zip(allocator.read_block(request, block), want):
            assert got.shape == (22, end - begin, 4, 64)
            assert (np.abs(got.cpu().double().numpy() - expected[:, begin:end]) <= 2.0**-11 * np.abs(expected[:, begin:end]) + 2.0**-25).all()
    pages = list(allocator.iter_layer_blocks(request, layer_index=7))
    assert [page[0].shape[0] for page in pages] == [16, 5]
    for kind in range(2):
        assert torch.equal(torch.cat([page[kind] for page in pages]), torch.cat([allocator.read_block(request, b)[kind][7] for b in range(2)]))


def test_attention_entry_points(device):
    allocator = _q4(device, 30)
    rng = np.random.default_rng(5)
    requests = []
    for i, length in enumerate((1, 40, 130)):
        request = RequestId(f"r{i}")
        allocator.create(KVReservation(request, 10))
        key, value = (torch.from_numpy(rng.standard_normal((22, length, 4, 64)).astype(np.float16)).to(device) for _ in range(2))
        allocator.append(request, key, value)
        requests.append(request)
    query = torch.from_numpy(rng.standard_normal((3, 32, 1, 64)).astype(np.float16)).to(device)
    out = paged_attention_batch(query, allocator, tuple(requests), layer_index=9)
    units = allocator.pool[9].cpu().numpy()
    for b, request in enumerate(requests):
        table = allocator.block_table(request)
        want, bound = ref.attention(query[b, :, 0].cpu().numpy(), units, table, allocator.cached_length(request))
        assert (np.abs(out[b, :, 0].cpu().double().numpy() - want) <= bound).all()
        alone = paged_attention(query[b : b + 1], allocator, request, layer_index=9)
        assert (np.abs(alone[0, :, 0].cpu().double().numpy() - want) <= bound).all()


class _Recorded(HipQ4Writer):
    """Keeps what each layer's write is given."""

    def __init__(self):
        super().__init__()
        self.rows = []

    def rope_append(self, pool, layer, qkv, rope_table, positions, slots, query_out):
        before = pool[layer].clone()
        rope = _hip.rope_kv_append_parts if qkv.ndim == 3 else _hip.rope_kv_append
        rows = torch.empty((2, 1, slots.shape[0], 4, 64), dtype=torch.float16, device=pool.device)
        query = torch.empty_like(query_out)
        rope(query, qkv, positions, rope_table, key_out=rows[0], value_out=rows[1])
        super().rope_append(pool, layer, qkv, rope_table, positions, slots, query_out)
        assert torch.equal(query.view(torch.int16), query_out.view(torch.int16))
        self.rows.append((rows.cpu().numpy(), slots.cpu().numpy(), before.cpu().numpy(), pool[layer].cpu().numpy()))


def test_decode_step_layer_by_layer(device, weights, monkeypatch):
    """Each layer writes its rotated key and its value, quantised, and attends to what the pool then stands for. (Logits are not
    compared with another evaluation's: a level may fall to either side of a border, and is a fifteenth of its row's range.)"""
    writer = _Recorded()
    allocator = KVAllocator(_q4(device).pool, kv_writer=writer)
    requests = tuple(_admit(allocator, weights, f"r{i}", _ids(device, n, 20 + i))[0] for i, n in enumerate((1, 15, 16, 49)))
    attended = []
    original = dec.attend_rows

    def attend(query, allocator, request_ids, layer):
        out, workspace = original(query, allocator, request_ids, layer)
        attended.append((query.cpu().numpy(), out.cpu().numpy(), allocator.pool[layer].cpu().numpy()))
        return out, workspace

    monkeypatch.setattr(dec, "attend_rows", attend)
    for step in range(2):
        writer.rows.clear()
        attended.clear()
        logits = dec.decode_paged(torch.tensor([[(7 * step + i) % 31] for i in range(4)], device=device), weights, allocator, requests)
        assert torch.isfinite(logits).all() and len(attended) == len(writer.rows) == 22
        for rows, slots, before, after in writer.rows:
            expected = before[None].copy()
            ref.write(expected, 0, rows[0], rows[1], slots)
            assert (after == expected[0]).all()
        for query, out, units in attended[::7]:
            for b, request in enumerate(requests):
                want, bound = ref.attention(query[b, :, 0], units, allocator.block_table(request), allocator.cached_length(request))
                assert (np.abs(out[b, :, 0].astype(np.float64) - want) <= bound).all()


@pytest.mark.parametrize("eight_bits", [False, True])
def test_graph_steps_equal_eager_ones(device, weights, eight_bits):
    if eight_bits:
        small = dec.quantize_weights(dec.random_weights(device=device, seed=11, layers=2, vocab=31, intermediate=32, norm_std=0.1))
        weights = dec.TinyLlamaWeights(small.embedding, small.layers * 11, small.final_norm, small.lm_head)
    eager, captured = _q4(device), _q4(device)
    requests = []
    for i, length in enumerate((1, 15, 16, 49, 100)):
        for allocator in (eager, captured):
            request, _ = _admit(allocator, weights, f"r{i}", _ids(device, length, 30 + i))
        requests.append(request)
    assert torch.equal(eager.pool, captured.pool)
    graph, padded = dec.DecodeGraph(weights, captured, 5), dec.DecodeGraph(weights, captured, 7)
    assert torch.equal(eager.pool, captured.pool)  # warm-up and capture wrote nothing
    for step in range(4):
        order = tuple(requests if step % 2 == 0 else reversed(requests))
        tokens = torch.tensor([[(5 * step + i) % 31] for i in range(5)], device=device)
        expected = dec.decode_paged(tokens, weights, eager, order)
        got = graph.step(tokens, order)
        graph.check_faults()
        assert torch.equal(got.view(torch.int16), expected.view(torch.int16))
        assert torch.equal(eager.pool, captured.pool)
    # Fewer requests than rows: nothing but their new slots changes.
    few = tuple(requests[1:4])
    before = captured.pool.clone()
    lengths = captured.cached_lengths(few)
    padded.step(torch.tensor([[1], [2], [3]], device=device), few)
    padded.check_faults()
    slots = [captured.block_table(r)[n // 16] * 16 + n % 16 for r, n in zip(few, lengths)]
    key, value = (torch.empty((22, 3, 4, 64), dtype=torch.float16, device=device) for _ in range(2))
    on = torch.tensor(slots, device=device)
    _hip.kv_read_q4(key, value, captured.pool, 0, on)
    assert torch.isfinite(key).all() and torch.isfinite(value).all()
    changed = (captured.pool != before).nonzero()
    places = np.zeros((40, 1152), dtype=bool)
    for slot in slots:
        block, t = divmod(slot, 16)
        for d in range(64):
            places[block, ref.key_place(t, d)[0]] = places[block, ref.value_place(t, d)[0]] = True
        for kind in range(2):
            places[block, ref.pair_place(kind, t) : ref.pair_place(kind, t) + 4] = True
    assert places[changed[:, 1].cpu().numpy(), changed[:, 3].cpu().numpy()].all()


def test_prefill_graph(device, weights):
    allocator, plain = _q4(device), _q4(device)
    graph = dec.PrefillGraph(weights, allocator, 64)
    for turn, length in enumerate((64, 1, 17, 50)):
        ids = _ids(device, length, 60 + turn)
        request = RequestId(f"p{turn}")
        allocator.create(KVReservation(request, 4))
        before = allocator.pool.clone()
        logits = graph.step(ids, request)
        _, expected = _admit(plain, weights, f"p{turn}", ids, spare=0)
        torch.testing.assert_close(logits[:, -1], expected[:, -1], atol=5e-3, rtol=5e-3)
        blocks = list(allocator.block_table(request))
        others = [b for b in range(40) if b not in blocks]
        assert torch.equal(allocator.pool[:, others], before[:, others])
        assert torch.isfinite(_rows(allocator, request)).all()
        plain.release_all(RequestId(f"p{turn}"))


def test_worker_tokens_equal_requests_alone(device, weights):
    rng = np.random.default_rng(8)
    requests = [
        GenerationRequest(RequestId(f"w{i}"), tuple(int(t) for t in rng.integers(3, 31, n)), max_new_tokens=m, ignore_eos=True)
        for i, (n, m) in enumerate(((3, 6), (17, 4), (30, 9), (16, 5), (1, 7)))
    ]
    worker = DecodeWorker(weights, _q4(device), max_active=3)
    for request in requests:
        worker.submit(request)
    finished = worker.run(max_steps=80)
    alone = _q4(device)
    for request in requests:
        ids = torch.tensor([request.input_ids], device=device)
        _, logits = _admit(alone, weights, str(request.request_id), ids)
        tokens = [int(logits[0, -1].argmax())]
        while len(tokens) < request.max_new_tokens:
            logits = dec.decode_paged(torch.tensor([[tokens[-1]]], device=device), weights, alone, (request.request_id,))
            tokens.append(int(logits[0, -1].argmax()))
        alone.release_all(request.request_id)
        assert finished[request.request_id].greedy_ids == tuple(tokens)
    worker = DecodeWorker(weights, _q4(device), max_active=3, graph_batch=(2, 4), prefill_graph_tokens=(16, 48))
    for request in requests:
        worker.submit(request)
    assert all(len(r.greedy_ids) == q.max_new_tokens for q, r in zip(requests, (worker.run(max_steps=80)[q.request_id] for q in requests)))


def test_allocated_pool(device):
    pool = allocate_kv_pool(PagedCoreConfig(kv_pool_mib=100, workspace_margin_mib=1), bits=4)
    assert pool.shape == (22, 100 * 2**20 // (22 * 4 * 1152), 4, 1152) and pool.dtype == torch.uint8
    allocator = KVAllocator(pool)
    assert allocator.quantized and allocator.capacity().total_blocks == pool.shape[1]
