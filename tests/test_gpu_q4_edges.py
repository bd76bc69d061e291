"""Decode attention over the 4-bit pool at the edges of fp16's range."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import q4_reference as ref
from pagedcore_amd import _hip
from tests.support import flags_clear

pytestmark = pytest.mark.gpu


def _attend(device, pool, layer, query, tables, lengths, new=(None, None), pad=False):
    lens, tabs = np.asarray(lengths, dtype=np.int32), np.asarray(tables, dtype=np.int32)
    plan = _hip.decode_plan(lens, tabs)
    if pad:
        full = np.zeros((_hip.plan_capacity(len(lens), tabs.shape[1]), plan.shape[1]), dtype=np.int32)
        full[: plan.shape[0]] = plan
        plan = full
    workspace = torch.zeros(_hip.workspace_bytes(len(lens), tabs.shape[1]), dtype=torch.uint8, device=device)
    out = torch.full((len(lens), 32, 64), 3.0, dtype=torch.float16, device=device)
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(device)  # noqa: E731
    _hip.planned_decode_attention_q4(out, query, pool, layer, up(lens), up(plan), tabs.shape[1], workspace, new_key=new[0], new_value=new[1])
    torch.cuda.synchronize()
    _hip.check_attention_faults(workspace, "test")
    assert flags_clear(workspace)
    return out


@pytest.mark.parametrize("length", [1, 15, 700])
@pytest.mark.parametrize("low", [0.0, -65504.0])
@pytest.mark.parametrize("fused", [False, True])
def test_steps_rounded_up_past_the_largest_value(device, length, low, fused):
    """Rows from `low` to 65504 have a step whose fifteenth multiple passes 65504 (65520 and 65536 in all). They are read as 65504,
    and tokens that all hold such a row attend to 65504 as well: no infinity comes of finite rows. A row of NaN stays NaN."""
    rng = np.random.default_rng(length)
    blocks = -(-length // 16)
    row = np.where(rng.integers(0, 2, (4, 64)) == 1, np.float16(65504), np.float16(low)).astype(np.float16)
    row[:, 0], row[:, 1] = low, 65504
    value = torch.from_numpy(row).to(device).expand(1, length, 4, 64).contiguous()
    key = torch.randn(1, length, 4, 64, dtype=torch.float16, device=device)
    pool = torch.zeros((22, blocks, 4, ref.UNIT), dtype=torch.uint8, device=device)
    slots = torch.arange(length, device=device)
    written = length - 1 if fused else length
    _hip.kv_append_q4(pool, 2, key[:, :written], value[:, :written], slots[:written])
    query = torch.randn(1, 32, 64, dtype=torch.float16, device=device)
    new = (key[0, -1:], value[0, -1:]) if fused else (None, None)
    tables = np.arange(blocks)[None]
    out = _attend(device, pool, 2, query, tables, [length], new)
    assert torch.equal(out[0].cpu(), torch.from_numpy(np.repeat(row, 8, axis=0)))
    back = torch.zeros_like(value)
    _hip.kv_read_q4(torch.zeros_like(key), back, pool, 2, slots)
    assert torch.equal(back, value)
    value[0, 0, 1, 3] = float("nan")
    _hip.kv_append_q4(pool, 2, key[:, :1], value[:, :1], slots[:1])
    out = _attend(device, pool, 2, query, tables, [length])
    assert torch.isnan(out[0, 8:16]).all() and torch.isfinite(out[0, :8]).all() and torch.isfinite(out[0, 16:]).all()


def test_a_row_given_for_both_is_the_values(device):
    key, value = (torch.randn(1, 1, 4, 64, dtype=torch.float16, device=device) for _ in range(2))
    pool = torch.zeros((22, 2, 4, ref.UNIT), dtype=torch.uint8, device=device)
    slots = torch.full((1,), 21, dtype=torch.int64, device=device)
    _hip.kv_append_q4(pool, 9, key, value, slots)
    both, rows = torch.zeros_like(key), [torch.zeros_like(key) for _ in range(2)]
    _hip.kv_read_q4(both, both, pool, 9, slots)
    _hip.kv_read_q4(*rows, pool, 9, slots)
    assert torch.equal(both, rows[1]) and not torch.equal(rows[0], rows[1])


def test_key_and_value_read_side_by_side(device):
    """K and V of a token next to each other, each a view of one buffer; one tensor for both is refused."""
    layers, tokens = 3, 40
    key, value = (torch.randn(layers, tokens, 4, 64, dtype=torch.float16, device=device) for _ in range(2))
    pool = torch.zeros((22, 3, 4, ref.UNIT), dtype=torch.uint8, device=device)
    slots = torch.arange(tokens, device=device)
    _hip.kv_append_q4(pool, 1, key, value, slots)
    apart = [torch.zeros_like(key) for _ in range(2)]
    _hip.kv_read_q4(*apart, pool, 1, slots)
    beside = torch.zeros((layers, tokens, 2, 4, 64), dtype=torch.float16, device=device)
    _hip.kv_read_q4(beside[:, :, 0], beside[:, :, 1], pool, 1, slots)
    assert torch.equal(beside, torch.stack(apart, dim=2))
    with pytest.raises(_hip.HipExtensionError, match="overlap"):
        _hip.kv_read_q4(key, key, pool, 1, slots)


def test_more_rows_than_a_launch_has_threads_for(device):
    """2^26 tokens and some, a row of 128 bytes at an odd address given for all of them (a token stride of 0): the first, the last and
    those around the middle are written, the others' slots lie outside the pool."""
    tokens, blocks = (1 << 26) + 37, 4
    rng = np.random.default_rng(2)
    rows = rng.standard_normal((2, 1, 1, 4, 64)).astype(np.float16)
    wide = torch.zeros(2, 257, dtype=torch.float16, device=device)
    wide[:, 1:] = torch.from_numpy(rows.reshape(2, 256)).to(device)
    key, value = (row[1:].view(1, 1, 4, 64).expand(1, tokens, 4, 64) for row in wide)
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=device)
    at = [0, 1, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26, tokens - 2, tokens - 1]
    places = [3, 17, 18, 40, 41, 42, 60, 63]
    slots[torch.tensor(at, device=device)] = torch.tensor(places, device=device)
    pool = torch.full((22, blocks, 4, ref.UNIT), 255, dtype=torch.uint8, device=device)
    expected = pool.cpu().numpy()
    _hip.kv_append_q4(pool, 6, key, value, slots)
    ref.write(expected, 6, *(np.repeat(x, len(at), axis=1) for x in rows), places)
    assert torch.equal(pool.cpu(), torch.from_numpy(expected))


@pytest.mark.parametrize("lengths", [[2000, 9, 700, 1500, 40], [4000], [1 + 97 * i % 2048 for i in range(30)], [5000, 300, 9000]])
@pytest.mark.parametrize("fused", [False, True])
def test_padding_a_plan_changes_no_bit(device, lengths, fused):
    """The same sequences behind the same tables, with the plan as it is and padded to its capacity with empty rows."""
    rng = np.random.default_rng(sum(lengths))
    need = -(-np.asarray(lengths) // 16)
    blocks = int(need.sum())
    tables, ids = np.zeros((len(lengths), max(300, int(need.max()))), dtype=np.int32), rng.permutation(blocks)
    for b, n in enumerate(need):
        tables[b, :n], ids = ids[:n], ids[n:]
    pool = torch.zeros((22, blocks, 4, ref.UNIT), dtype=torch.uint8, device=device)
    rows = [torch.randn(1, blocks * 16, 4, 64, dtype=torch.float16, device=device) for _ in range(2)]
    _hip.kv_append_q4(pool, 8, *rows, torch.arange(blocks * 16, device=device))
    query = torch.randn(len(lengths), 32, 64, dtype=torch.float16, device=device)
    new = tuple(torch.randn(len(lengths), 4, 64, dtype=torch.float16, device=device) for _ in range(2)) if fused else (None, None)
    plain, padded = (_attend(device, pool, 8, query, tables, lengths, new, pad) for pad in (False, True))
    assert torch.equal(plain.view(torch.int16), padded.view(torch.int16)), (plain != padded).flatten(1).any(1).nonzero().flatten().tolist()
