"""Decode attention over the 4-bit pool, held to a bound near fp16's rounding: large queries, scores that rise, and the kernel that
a serving batch takes, over bins of many blocks."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import q4_reference as ref
from pagedcore_amd import _hip
from tests.q4_cases import CASES, build
from tests.support import flags_clear

pytestmark = pytest.mark.gpu


def _attend(device, pool, layer, query, tables, lengths, new=(None, None)):
    lens, tabs = np.asarray(lengths, dtype=np.int32), np.ascontiguousarray(tables, dtype=np.int32)
    plan = _hip.decode_plan(lens, tabs)
    workspace = torch.zeros(_hip.workspace_bytes(len(lens), tabs.shape[1]), dtype=torch.uint8, device=device)
    out = torch.full((len(lens), 32, 64), 3.0, dtype=torch.float16, device=device)
    _hip.planned_decode_attention_q4(
        out, query, pool, layer, torch.from_numpy(lens).to(device), torch.from_numpy(plan).to(device), tabs.shape[1], workspace,
        new_key=new[0], new_value=new[1],
    )
    torch.cuda.synchronize()
    _hip.check_attention_faults(workspace, "test")
    assert flags_clear(workspace)
    return out, int(plan[:, 1].max())


def _check(out, query, units, tables, lengths, rows=None):
    worst = 0.0
    for b in range(len(lengths)) if rows is None else rows:
        want, bound = ref.close_attention(query[b], units, tables[b], int(lengths[b]))
        off = np.abs(out[b].cpu().double().numpy() - want) / bound
        assert (off <= 1.0).all(), f"row {b} of length {lengths[b]}: {off.max():.3g} of the bound, heads {sorted(set(np.nonzero(off > 1)[0].tolist()))}"
        worst = max(worst, off.max())
    print(f"{worst:.3g} of the bound at most")


SERVING = [1, 64, 65, 130, 2048, 333, 700, 17, 1000, 1500, 48, 900]  # more than eight sequences: two waves a kv head


@pytest.mark.parametrize("lengths", ["few", "serving"])
@pytest.mark.parametrize("case", list(CASES))
def test_attention(device, case, lengths):
    query, units, tables, lengths = build(case, None if lengths == "few" else SERVING)
    pool = torch.zeros((22, *units.shape), dtype=torch.uint8, device=device)
    pool[11] = torch.from_numpy(units).to(device)
    out, _ = _attend(device, pool, 11, torch.from_numpy(query).to(device), tables, lengths)
    _check(out, query, units, tables, lengths)


def _batch(device, lengths, layer, seed):
    """A pool with random rows in every slot of a layer, and the queries and tables of sequences in scattered blocks."""
    rng = np.random.default_rng(seed)
    need = -(-np.asarray(lengths) // 16)
    blocks = int(need.sum())
    ids, tables = rng.permutation(blocks), np.zeros((len(lengths), int(need.max())), dtype=np.int32)
    tables[np.arange(tables.shape[1]) < need[:, None]] = ids
    pool = torch.empty((22, blocks, 4, ref.UNIT), dtype=torch.uint8, device=device)
    gen = torch.Generator(device=device).manual_seed(seed)
    for at in range(0, blocks, 4096):
        slots = torch.arange(16 * at, 16 * min(at + 4096, blocks), device=device)
        key, value = (torch.randn(1, slots.shape[0], 4, 64, dtype=torch.float16, device=device, generator=gen) for _ in range(2))
        _hip.kv_append_q4(pool, layer, key, value, slots)
    query = torch.randn(len(lengths), 32, 64, dtype=torch.float16, device=device, generator=gen)
    return pool, query, tables


@pytest.mark.parametrize("lengths,longest,rows", [
    ([1 + 331 * i % 2048 for i in range(64)], 16, None),  # a ragged serving batch
    ([2048] * 64, 32, range(0, 64, 9)),
    ([2048] * 256, 128, range(0, 256, 51)),
    ([2041] * 600, 253, range(0, 600, 99)),
    ([1 + 57 * i % 64 for i in range(256)], 8, range(0, 256, 5)),  # many short sequences
], ids=["64 ragged", "64 x 2048", "256 x 2048", "600 x 2041", "256 short"])
def test_serving_batches(device, lengths, longest, rows):
    pool, query, tables = _batch(device, lengths, 4, len(lengths))
    out, blocks = _attend(device, pool, 4, query, tables, lengths)
    assert blocks >= longest
    _check(out, query.cpu().numpy(), pool[4].cpu().numpy(), tables, lengths, rows)


@pytest.mark.parametrize("lengths", [[1 + 331 * i % 2048 for i in range(64)], [2048] * 256], ids=["64 ragged", "256 x 2048"])
def test_fused_append_of_a_serving_batch(device, lengths):
    pool, query, tables = _batch(device, lengths, 7, 5)
    new = [torch.randn(len(lengths), 4, 64, dtype=torch.float16, device=device) for _ in range(2)]
    pair = pool.clone()
    last = np.asarray(lengths) - 1
    slots = tables[np.arange(len(lengths)), last // 16].astype(np.int64) * 16 + last % 16
    _hip.kv_append_q4(pair, 7, new[0][None], new[1][None], torch.from_numpy(slots).to(device))
    expected, _ = _attend(device, pair, 7, query, tables, lengths)
    out, _ = _attend(device, pool, 7, query, tables, lengths, new)
    assert torch.equal(out.view(torch.int16), expected.view(torch.int16))
    assert torch.equal(pool[7], pair[7])


@pytest.mark.parametrize("lengths", [SERVING, [2041] * 600], ids=["12 ragged", "600 x 2041"])
def test_block_ids_outside_the_pool_of_a_serving_batch(device, lengths):
    """Whichever wave and whichever of its blocks they belong to: their sequence is NaN, the others keep their bits."""
    pool, query, tables = _batch(device, lengths, 2, 9)
    clean, _ = _attend(device, pool, 2, query, tables, lengths)
    lens = np.asarray(lengths, dtype=np.int32)
    broken, hit = tables.copy(), []
    for b in range(1, len(lengths), 5):
        blocks = -(-lengths[b] // 16)
        broken[b, (0, blocks - 1, blocks // 2, 63, 64, 65, 100)[b // 5 % 7] % blocks] = (pool.shape[1], -1, 1 << 30)[b // 5 % 3]
        hit.append(b)
    plan = torch.from_numpy(_hip.decode_plan(lens, broken)).to(device)
    workspace = torch.zeros(_hip.workspace_bytes(len(lens), tables.shape[1]), dtype=torch.uint8, device=device)
    out = torch.zeros_like(query)
    _hip.planned_decode_attention_q4(out, query, pool, 2, torch.from_numpy(lens).to(device), plan, tables.shape[1], workspace)
    torch.cuda.synchronize()
    with pytest.raises(_hip.AttentionFaultError, match="block id"):
        _hip.check_attention_faults(workspace, "test")
    others = [b for b in range(len(lengths)) if b not in hit]
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[others].view(torch.int16), clean[others].view(torch.int16))
