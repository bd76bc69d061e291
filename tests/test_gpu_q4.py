"""The 4-bit KV pool on the GPU: appended bytes equal the definition's bit for bit, rows read back are its values rounded
once, attention stays within a bound derived from its operations, the fused append equals the pair of calls."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import q4_reference as ref
from pagedcore_amd import _hip
from pagedcore_amd.decoder import capture_graph
from tests.support import fault_word, flags_clear, workspace_flags

pytestmark = pytest.mark.gpu


def _rows(rng, *shape):
    """K or V rows float16 [..., 4, 64] of several scales, some constant, some with ties."""
    x = rng.standard_normal((*shape, 4, 64)) * 2.0 ** rng.integers(-6, 4, (*shape, 4, 1)) + rng.standard_normal((*shape, 4, 1))
    x = x.astype(np.float16)
    flat = x.reshape(-1, 64)
    flat[3::17] = flat[3::17, :1]  # constant rows
    flat[5::13] = np.float16(0.5) * rng.integers(-16, 16, flat[5::13].shape)  # whole halves: many ties
    return x


def _pool(rng, blocks):
    return rng.integers(0, 256, (22, blocks, 4, ref.UNIT), dtype=np.uint8)


def _up(array, device):
    return torch.from_numpy(np.ascontiguousarray(array)).to(device)


def _tables(rng, lengths, spare=3):
    need = -(-np.asarray(lengths) // 16)
    blocks = int(need.sum()) + spare
    ids = rng.permutation(blocks).astype(np.int32)
    tables = np.zeros((len(lengths), max(1, int(need.max()))), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = ids[at : at + n]
        at += n
    return tables, blocks


def _filled(rng, blocks, layer):
    """A pool whose layer holds quantised rows in every slot, other bytes random (whatever they stand for)."""
    pool = _pool(rng, blocks)
    key, value = _rows(rng, 1, blocks * 16), _rows(rng, 1, blocks * 16)
    ref.write(pool, layer, key, value, range(blocks * 16))
    return pool


def _written(rng, blocks, layer, device):
    """The same, on the device and quantised there, where no definition is compared with."""
    pool = torch.randint(0, 256, (22, blocks, 4, ref.UNIT), dtype=torch.uint8, device=device)
    key, value = (_up(rng.standard_normal((1, blocks * 16, 4, 64)).astype(np.float16), device) for _ in range(2))
    _hip.kv_append_q4(pool, layer, key, value, torch.arange(blocks * 16, device=device))
    return pool


@pytest.mark.parametrize("layers,begin,tokens,start", [(1, 21, 1, 0), (22, 0, 17, 5), (3, 7, 64, 0), (2, 20, 131, 15), (5, 0, 4, 2), (22, 0, 27, 7), (1, 4, 700, 0)])
def test_append_bytes(device, layers, begin, tokens, start):
    rng = np.random.default_rng(tokens)
    blocks = -(-(start + tokens) // 16) + 2
    table = rng.permutation(blocks)
    at = np.arange(start, start + tokens)
    slots = table[at // 16] * 16 + at % 16
    pool = _pool(rng, blocks)
    key, value = _rows(rng, layers, tokens), _rows(rng, layers, tokens)
    expected = pool.copy()
    ref.write(expected, begin, key, value, slots)
    got = _up(pool, device)
    _hip.kv_append_q4(got, begin, _up(key, device), _up(value, device), _up(slots, device))
    assert torch.equal(got.cpu(), torch.from_numpy(expected))


@pytest.mark.parametrize("offset", [0, 8, 1])
def test_append_strided_and_skipped(device, offset):
    """Rows as views of wider ones (16-byte aligned or not), slots in any order, some outside the pool."""
    rng = np.random.default_rng(7)
    tokens, blocks = 50, 6
    wide = np.zeros((2, tokens, 600 + offset), dtype=np.float16)
    wide[:, :, offset : offset + 256] = _rows(rng, 2, tokens).reshape(2, tokens, 256)
    wide[:, :, offset + 256 : offset + 512] = _rows(rng, 2, tokens).reshape(2, tokens, 256)
    slots = rng.permutation(blocks * 16)[:tokens].astype(np.int64)
    slots[[3, 11, 12]] = (-1, blocks * 16, 1 << 40)
    pool = _pool(rng, blocks)
    on = _up(wide, device)
    key, value = (on[:, :, at : at + 256].unflatten(-1, (4, 64)) for at in (offset, offset + 256))
    got = _up(pool, device)
    _hip.kv_append_q4(got, 4, key, value, _up(slots, device))
    expected = pool.copy()
    ref.write(expected, 4, key.cpu().numpy(), value.cpu().numpy(), slots)
    assert torch.equal(got.cpu(), torch.from_numpy(expected))
    # Read back into views of the same alignment; skipped tokens' rows keep what they held.
    back = torch.full((2, 2, tokens, 600 + offset), 7.0, dtype=torch.float16, device=device)
    rows = [back[i, :, :, offset : offset + 256].unflatten(-1, (4, 64)) for i in range(2)]
    _hip.kv_read_q4(rows[0], rows[1], got, 4, _up(slots, device))
    inside = (slots >= 0) & (slots < blocks * 16)
    for kind in range(2):
        want = np.stack([ref.rows(expected[4 + layer], kind, np.where(inside, slots, 0)) for layer in range(2)])
        _assert_read(rows[kind].cpu().numpy()[:, inside], want[:, inside])
        assert (rows[kind].cpu().numpy()[:, ~inside] == 7.0).all()
    back[..., offset : offset + 256] = 7.0
    assert (back == 7.0).all()


@pytest.mark.parametrize("kind", ["start_0", "start_8", "start_13", "backwards", "holes", "swapped", "across"])
@pytest.mark.parametrize("offset", [0, 3])
def test_prompt_rows(device, kind, offset):
    """Enough rows that eight tokens go together where their slots do: whole halves of blocks, halves cut at both ends, slots in
    another order, tokens that are skipped; rows as views of wider ones, aligned to 16 bytes or not."""
    rng = np.random.default_rng(len(kind))
    layers, tokens = 4, 203
    table = rng.permutation(16)
    at = np.arange({"start_8": 8, "start_13": 13}.get(kind, 0), 240)[:tokens]
    slots = (table[at // 16] * 16 + at % 16).astype(np.int64)
    if kind == "backwards":
        slots = slots[::-1].copy()
    elif kind == "holes":
        slots[[0, 9, 63, 64, 100, 202]] = (-1, 256, -5, 1 << 33, -1, 300)
    elif kind == "swapped":
        slots[[16, 17]], slots[[40, 48]] = slots[[17, 16]], slots[[48, 40]]
    elif kind == "across":  # consecutive slots that go on from one block into the next
        slots = np.arange(4, 4 + tokens, dtype=np.int64)
    wide = np.zeros((2, layers, tokens, 264 + offset), dtype=np.float16)
    wide[..., offset : offset + 256] = _rows(rng, 2, layers, tokens).reshape(2, layers, tokens, 256)
    on = _up(wide, device)
    key, value = (on[i, ..., offset : offset + 256].unflatten(-1, (4, 64)) for i in range(2))
    pool = _pool(rng, 16)
    expected = pool.copy()
    ref.write(expected, 9, key.cpu().numpy(), value.cpu().numpy(), slots)
    got = _up(pool, device)
    _hip.kv_append_q4(got, 9, key, value, _up(slots, device))
    assert torch.equal(got.cpu(), torch.from_numpy(expected))
    back = torch.full((2, layers, tokens, 264 + offset), 7.0, dtype=torch.float16, device=device)
    rows = [back[i, ..., offset : offset + 256].unflatten(-1, (4, 64)) for i in range(2)]
    _hip.kv_read_q4(rows[0], rows[1], got, 9, _up(slots, device))
    inside = (slots >= 0) & (slots < 256)
    for i in range(2):
        want = np.stack([ref.rows(expected[9 + layer], i, np.where(inside, slots, 0)) for layer in range(layers)])
        _assert_read(rows[i].cpu().numpy()[:, inside], want[:, inside])
        assert (rows[i].cpu().numpy()[:, ~inside] == 7.0).all()
    back[..., offset : offset + 256] = 7.0
    assert (back == 7.0).all()


def _assert_read(got, want):
    """One rounding to fp16 behind one to fp32 (half steps 2^-11 and 2^-24 of the value; 2^-25 below fp16's normal range); what
    lies past fp16's largest value is that value."""
    want = np.minimum(want, 65504.0)
    fine = np.isfinite(want)
    assert (np.isnan(got) == ~fine).all()
    off = np.abs(got.astype(np.float64) - want)[fine]
    assert (off <= (2.0**-11 + 2.0**-23) * np.abs(want[fine]) + 2.0**-25).all()


@pytest.mark.parametrize("layers,begin,tokens", [(1, 3, 1), (22, 0, 20), (22, 0, 33), (2, 20, 300)])
def test_read_rows(device, layers, begin, tokens):
    rng = np.random.default_rng(tokens)
    blocks = tokens // 16 + 3
    pool = _pool(rng, blocks)
    for layer in range(layers):
        ref.write(pool, begin + layer, _rows(rng, 1, blocks * 16), _rows(rng, 1, blocks * 16), range(blocks * 16))
    slots = rng.integers(0, blocks * 16, tokens)  # a slot may be read twice
    key = torch.zeros((layers, tokens, 4, 64), dtype=torch.float16, device=device)
    value = torch.zeros_like(key)
    _hip.kv_read_q4(key, value, _up(pool, device), begin, _up(slots, device))
    for kind, got in enumerate((key, value)):
        _assert_read(got.cpu().numpy(), np.stack([ref.rows(pool[begin + layer], kind, slots) for layer in range(layers)]))


def test_a_row_is_the_same_whichever_call_writes_or_reads_it(device):
    """Eight tokens a wave, a token a wave, rows aligned to 16 bytes or not: the same bytes and the same values bit for bit."""
    rng = np.random.default_rng(18)
    layers, tokens, blocks = 3, 2048, 128
    key, value = (_up(rng.standard_normal((layers, tokens, 4, 64)).astype(np.float16), device) for _ in range(2))
    slots = torch.arange(tokens, device=device)
    pools = [torch.zeros((22, blocks, 4, ref.UNIT), dtype=torch.uint8, device=device) for _ in range(3)]
    wide = torch.empty((2, layers, tokens, 4 * 64 + 1), dtype=torch.float16, device=device)
    odd = [x[..., 1:].unflatten(-1, (4, 64)) for x in wide]
    odd[0].copy_(key)
    odd[1].copy_(value)
    _hip.kv_append_q4(pools[0], 0, key, value, slots)
    _hip.kv_append_q4(pools[1], 0, *odd, slots)
    back = torch.zeros((2, layers, tokens, 4, 64), dtype=torch.float16, device=device)
    _hip.kv_read_q4(back[0], back[1], pools[0], 0, slots)
    for at in range(0, tokens, 100):
        some = slice(at, at + 100)
        _hip.kv_append_q4(pools[2], 0, key[:, some], value[:, some], slots[some])
        part = torch.zeros_like(back[:, :, some])
        _hip.kv_read_q4(part[0], part[1], pools[0], 0, slots[some])
        assert torch.equal(part.view(torch.int16), back[:, :, some].view(torch.int16))
    assert torch.equal(pools[0], pools[1]) and torch.equal(pools[0], pools[2])
    wide.zero_()
    _hip.kv_read_q4(*odd, pools[0], 0, slots)
    assert all(torch.equal(x, y) for x, y in zip(odd, back))


def test_rows_of_every_kind(device):
    """Infinities and NaN, the widest and the narrowest spans, subnormal steps, zeros of both signs."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 16, 4, 64)).astype(np.float16)
    f = x.reshape(-1, 64)
    f[0], f[1, 5], f[2, 63], f[3, :2] = np.nan, np.inf, -np.inf, (np.inf, -np.inf)
    f[4], f[5] = 65504, np.where(np.arange(64) % 2, 65504, -65504)
    f[6] = np.where(np.arange(64) % 2, -0.0, 0.0)
    f[7] = (np.arange(64) % 23) * np.float16(2.0**-24)  # a span whose fifteenth lies between two subnormals
    f[8] = (np.arange(64) % 16) * np.float16(2.0**-24)
    f[9] = np.arange(64) * np.float16(2.0**-14)
    f[10] = np.where(np.arange(64) == 17, 2.0**-24, 0)
    f[11] = -(np.arange(64).astype(np.float16))
    pool = _pool(rng, 2)
    expected = pool.copy()
    ref.write(expected, 0, x, x[..., ::-1].copy(), range(16))
    got = _up(pool, device)
    slots = torch.arange(16, device=device)
    _hip.kv_append_q4(got, 0, _up(x, device), _up(x[..., ::-1], device), slots)
    key = torch.zeros((1, 16, 4, 64), dtype=torch.float16, device=device)
    value = torch.zeros_like(key)
    _hip.kv_read_q4(key, value, got, 0, slots)
    got = got.cpu().numpy()
    bad = [i for i in range(64) if not np.isfinite(f[i]).all()]
    for kind, rows in enumerate((key, value)):
        want = ref.rows(expected[0], kind, np.arange(16))
        _assert_read(rows.cpu().numpy()[0], want)
        assert np.isnan(rows.cpu().numpy()[0].reshape(-1, 64)[bad]).all()
    assert (got == expected).all()


@pytest.mark.parametrize("tokens", [3, 1200])
def test_rows_of_zeros_have_the_bytes_of_zero(device, tokens):
    """Rows of -0 alone, of both zeros, of +0: all of them a minimum and a step of +0. (-0 less +0 is -0, which must not become the step.)"""
    x = np.zeros((4, tokens, 4, 64), dtype=np.float16)
    x[:, ::3] = -0.0
    x[:, 1::3, :, ::2] = -0.0
    slots = torch.arange(tokens, device=device)
    pool = torch.full((22, tokens // 16 + 1, 4, ref.UNIT), 255, dtype=torch.uint8, device=device)
    expected = pool.cpu().numpy()
    ref.write(expected, 2, x, x, range(tokens))
    _hip.kv_append_q4(pool, 2, _up(x, device), _up(x, device), slots)
    assert torch.equal(pool.cpu(), torch.from_numpy(expected))


def _attend(device, pool, layer, query, tables, lengths, new=None, out=None, workspace=None):
    batch = len(lengths)
    lens, tabs = np.asarray(lengths, dtype=np.int32), np.asarray(tables, dtype=np.int32)
    plan = _up(_hip.decode_plan(lens, tabs), device)
    if workspace is None:
        workspace = torch.zeros(_hip.workspace_bytes(batch, tabs.shape[1]), dtype=torch.uint8, device=device)
    if out is None:
        out = torch.full((batch, 32, 64), 3.0, dtype=torch.float16, device=device)
    key, value = new if new is not None else (None, None)
    _hip.planned_decode_attention_q4(out, query, pool, layer, _up(lens, device), plan, tabs.shape[1], workspace, new_key=key, new_value=value)
    torch.cuda.synchronize()
    _hip.check_attention_faults(workspace, "test")
    assert flags_clear(workspace)
    return out


def _check_rows(out, query, units, tables, lengths, rows=None):
    got = out.cpu().numpy().astype(np.float64)
    q = query.cpu().numpy()
    for b in range(len(lengths)) if rows is None else rows:
        if lengths[b] == 0:
            assert (got[b] == 3.0).all()  # left as it was
            continue
        want, bound = ref.attention(q[b], units, tables[b], int(lengths[b]))
        off = np.abs(got[b] - want)
        assert (off <= bound).all(), f"row {b} of length {lengths[b]}: {np.max(off / bound):.3g} of the bound"


CASES = {
    "one": [1],
    "short": [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65],
    "block_ends": [128, 127, 129, 112, 80, 96, 16, 64],
    "with_empty_rows": [0, 5, 0, 200, 0],
    "cut": [2048, 3, 1500, 700],
    "long": [9001],
    "long_ragged": [5000, 4097, 1, 0, 12003, 17, 8191],
    "group_of_32": [4000],
    "long_few": [8191, 9, 5000],
    "many_short": [1 + i % 48 for i in range(300)],
}


@pytest.mark.parametrize("name", list(CASES))
def test_attention(device, name):
    rng = np.random.default_rng(len(name))
    lengths = CASES[name]
    tables, blocks = _tables(rng, lengths)
    layer = 5
    pool = _filled(rng, blocks, layer)
    # Slots past a length hold anything, rows of NaN among it.
    for b, n in enumerate(lengths):
        if n % 16:
            unit = pool[layer, tables[b, n // 16]]
            for t in range(n % 16, 16):
                for kind in range(2):
                    at = ref.pair_place(kind, t)
                    unit[:, at : at + 4] = np.frombuffer(np.array([np.nan, np.inf], dtype=np.float16).tobytes(), dtype=np.uint8)
    query = _up(rng.standard_normal((len(lengths), 32, 64)).astype(np.float16), device)
    out = _attend(device, _up(pool, device), layer, query, tables, lengths)
    rows = range(0, len(lengths), 7) if len(lengths) > 100 else None
    _check_rows(out, query, pool[layer], tables, lengths, rows)


@pytest.mark.parametrize("scale", [0.0, 2.0**-20, 30.0, 1000.0, 20000.0])
def test_attention_of_sharp_and_flat_scores(device, scale):
    rng = np.random.default_rng(3)
    lengths = [77, 400]
    tables, blocks = _tables(rng, lengths)
    pool = _filled(rng, blocks, 0)
    query = _up(np.clip(rng.standard_normal((2, 32, 64)) * scale, -65504, 65504).astype(np.float16), device)
    out = _attend(device, _up(pool, device), 0, query, tables, lengths)
    _check_rows(out, query, pool[0], tables, lengths)


@pytest.mark.parametrize("exponent", [-24, -20, -14, 12])
def test_attention_over_rows_of_tiny_and_large_steps(device, exponent):
    """Steps that are fp16 subnormals (down to the smallest) and steps and minima of thousands."""
    rng = np.random.default_rng(8)
    lengths = [77, 1000, 3]
    tables, blocks = _tables(rng, lengths)
    pool = _pool(rng, blocks)
    key, value = (np.clip(rng.standard_normal((1, blocks * 16, 4, 64)) * 2.0**exponent, -60000, 60000).astype(np.float16) for _ in range(2))
    ref.write(pool, 4, key, value, range(blocks * 16))
    query = _up((rng.standard_normal((3, 32, 64)) * (30 if exponent < 0 else 2.0**-8)).astype(np.float16), device)
    out = _attend(device, _up(pool, device), 4, query, tables, lengths)
    _check_rows(out, query, pool[4], tables, lengths)


def test_constant_values_come_back_exactly(device):
    rng = np.random.default_rng(4)
    lengths = [333, 16]
    tables, blocks = _tables(rng, lengths)
    pool = _pool(rng, blocks)
    value = np.full((1, blocks * 16, 4, 64), 3.140625, dtype=np.float16)
    ref.write(pool, 2, _rows(rng, 1, blocks * 16), value, range(blocks * 16))
    query = _up(rng.standard_normal((2, 32, 64)).astype(np.float16), device)
    out = _attend(device, _up(pool, device), 2, query, tables, lengths)
    assert (out == 3.140625).all()


def test_nan_rows_stay_in_their_head_and_sequence(device):
    rng = np.random.default_rng(5)
    lengths = [40, 70, 90]
    tables, blocks = _tables(rng, lengths)
    pool = _filled(rng, blocks, 1)
    query = rng.standard_normal((3, 32, 64)).astype(np.float16)
    query[2, 9] = np.nan
    on = _up(pool, device)
    clean = _attend(device, on, 1, _up(query, device), tables, lengths)
    x = _rows(rng, 1, 2)
    x[0, 0, 2, 7], x[0, 1, 3, 0] = np.nan, np.inf
    fine = _rows(rng, 1, 2)
    slots = np.array([tables[1, 33 // 16] * 16 + 33 % 16, tables[0, 5 // 16] * 16 + 5 % 16], dtype=np.int64)
    _hip.kv_append_q4(on, 1, _up(x, device), _up(fine, device), _up(slots, device))
    out = _attend(device, on, 1, _up(query, device), tables, lengths)
    nan = torch.isnan(out).all(-1).cpu()
    assert (torch.isnan(out).any(-1).cpu() == nan).all()
    expected = torch.zeros((3, 32), dtype=torch.bool)
    expected[1, 16:24] = expected[0, 24:32] = expected[2, 9] = True
    assert torch.equal(nan, expected)
    assert torch.equal(out[2, :9].view(torch.int16), clean[2, :9].view(torch.int16))


@pytest.mark.parametrize("lengths", [[50, 300, 20], [50, 9000, 20]])
def test_block_ids_outside_the_pool(device, lengths):
    rng = np.random.default_rng(6)
    tables, blocks = _tables(rng, lengths)
    pool = _written(rng, blocks, 0, device)
    query = _up(rng.standard_normal((3, 32, 64)).astype(np.float16), device)
    clean = _attend(device, pool, 0, query, tables, lengths)
    for bad in (blocks, -1, 1 << 30):
        broken = tables.copy()
        broken[1, 7] = bad
        lens = np.array(lengths, dtype=np.int32)
        workspace = torch.zeros(_hip.workspace_bytes(3, tables.shape[1]), dtype=torch.uint8, device=device)
        out = torch.zeros_like(query)
        _hip.planned_decode_attention_q4(out, query, pool, 0, _up(lens, device), _up(_hip.decode_plan(lens, broken), device), tables.shape[1], workspace)
        torch.cuda.synchronize()
        with pytest.raises(_hip.AttentionFaultError, match="block id"):
            _hip.check_attention_faults(workspace, "test")
        assert torch.isnan(out[1]).all()
        assert torch.equal(out[[0, 2]].view(torch.int16), clean[[0, 2]].view(torch.int16))


@pytest.mark.parametrize("name", ["one", "short", "block_ends", "cut", "many_short", "with_empty_rows", "long_ragged", "long_few"])
def test_fused_append_equals_the_pair(device, name):
    rng = np.random.default_rng(10 + len(name))
    lengths = CASES[name]
    tables, blocks = _tables(rng, lengths)
    layer = 20
    pool = _written(rng, blocks, layer, device)
    query = _up(rng.standard_normal((len(lengths), 32, 64)).astype(np.float16), device)
    new = [_up(_rows(rng, len(lengths)), device) for _ in range(2)]
    slots = np.array([tables[b, (n - 1) // 16] * 16 + (n - 1) % 16 if n else -1 for b, n in enumerate(lengths)], dtype=np.int64)
    pair = pool.clone()
    _hip.kv_append_q4(pair, layer, new[0][None], new[1][None], _up(slots, device))
    expected = _attend(device, pair, layer, query, tables, lengths)
    for _ in range(2):  # a second call writes the same bytes
        out = _attend(device, pool, layer, query, tables, lengths, new)
        assert torch.equal(out.view(torch.int16), expected.view(torch.int16))
        assert torch.equal(pool, pair)


def _spans(plan):
    """Of every cut sequence its parts: {part: (plan row, segment)}."""
    spans = {}
    for row in range(plan.shape[0]):
        for s in range(int(plan[row, 0])):
            b, _, _, _, _, part, parts, _ = (int(v) for v in plan[row, 8 + 8 * s : 16 + 8 * s])
            if parts > 1:
                spans.setdefault(b, {})[part] = (row, s)
    return spans


@pytest.mark.parametrize("fault", ["first part", "part that folds", "last part", "slots outside the workspace", "sequence outside the batch"])
@pytest.mark.parametrize("lengths", [[300, 40, 2048, 1500], [4000], [40, 9000, 700], [300, 40, 2048, 1500, 1, 64, 7, 900, 30, 5], [40, 9000, 12000, 700]])
def test_plans_that_do_not_match(device, lengths, fault):
    """A plan without one of a cut sequence's parts: the fold waits for it a bounded time, its row is NaN and the fault is
    reported; without the last part, or with its partials outside the workspace, or under another number, its row is left alone.
    Rows that the change does not touch keep their bits, and the next call on the workspace is right."""
    rng = np.random.default_rng(16)
    tables, blocks = _tables(rng, lengths)
    lens, layer, width = np.asarray(lengths, dtype=np.int32), 7, tables.shape[1]
    pool = _written(rng, blocks, layer, device)
    query = _up(rng.standard_normal((len(lengths), 32, 64)).astype(np.float16), device)
    workspace = torch.zeros(_hip.workspace_bytes(len(lengths), width), dtype=torch.uint8, device=device)
    good = _attend(device, pool, layer, query, tables, lengths, workspace=workspace)
    plan = _hip.decode_plan(lens, tables)
    spans = _spans(plan)
    b = int(np.argmax(lens))
    parts = spans[b]
    last = max(parts)
    nan_rows, left_alone = set(), {b}
    if fault in ("first part", "part that folds", "last part"):
        row = parts[{"first part": 0, "part that folds": min(7, last - 1), "last part": last}[fault]][0]
        inside = {int(x) for x in plan[row, 8 : 8 + 8 * int(plan[row, 0]) : 8]}
        nan_rows = {x for x in inside if x in spans and spans[x][max(spans[x])][0] != row}
        left_alone = inside - nan_rows
        plan[row] = 0
    elif fault == "slots outside the workspace":
        for row, s in parts.values():
            plan[row, 8 + 8 * s + 7] = 1 << 30
    else:
        for row, s in parts.values():
            plan[row, 8 + 8 * s] = len(lengths) + 5
    out = torch.full_like(good, 3.0)
    _hip.planned_decode_attention_q4(out, query, pool, layer, _up(lens, device), _up(plan, device), width, workspace)
    torch.cuda.synchronize()
    for x in range(len(lengths)):
        if x in nan_rows:
            assert torch.isnan(out[x]).all(), x
        elif x in left_alone:
            assert (out[x] == 3.0).all(), x
        else:
            assert torch.equal(out[x].view(torch.int16), good[x].view(torch.int16)), x
    assert fault_word(workspace) == (_hip.FAULT_MERGE_TIMEOUT if nan_rows else 0)
    if nan_rows:
        with pytest.raises(_hip.AttentionFaultError, match="bounded wait"):
            _hip.check_attention_faults(workspace, "test")
    elif fault == "last part":
        assert workspace_flags(workspace).any()
    again = _attend(device, pool, layer, query, tables, lengths, workspace=workspace)
    assert torch.equal(again.view(torch.int16), good.view(torch.int16))


def test_two_graphs_share_a_workspace(device):
    """Graphs of two layers' attention, replayed in turn on one stream over one workspace, and a plan padded to its capacity."""
    rng = np.random.default_rng(17)
    lengths = [2000, 9, 700, 4500]
    tables, blocks = _tables(rng, lengths)
    width = tables.shape[1]
    lens = _up(np.asarray(lengths, dtype=np.int32), device)
    pool = _written(rng, blocks, 0, device)
    pool[1] = pool[0].flip(0)
    host = np.zeros((_hip.plan_capacity(len(lengths), width), _hip.load().pc_attn_plan_record_ints()), dtype=np.int32)
    _hip.decode_plan_into(np.asarray(lengths, dtype=np.int32), tables, host)
    plan = _up(host, device)
    workspace = torch.zeros(_hip.workspace_bytes(len(lengths), width), dtype=torch.uint8, device=device)
    query = torch.zeros((len(lengths), 32, 64), dtype=torch.float16, device=device)
    runs = []
    for layer in (0, 1):

        def step(layer=layer):
            out = torch.zeros_like(query)
            _hip.planned_decode_attention_q4(out, query, pool, layer, lens, plan, width, workspace)
            return out

        runs.append(capture_graph(step, device))
    for turn in range(3):
        query.copy_(torch.from_numpy(rng.standard_normal(tuple(query.shape)).astype(np.float16)))
        for graph, _ in runs:
            graph.replay()
        for layer, (_, out) in enumerate(runs):
            expected = _attend(device, pool, layer, query, tables, lengths)
            assert torch.equal(out.view(torch.int16), expected.view(torch.int16))
    _hip.check_attention_faults(workspace, "test")
    assert flags_clear(workspace)


def test_decode_steps_in_a_graph(device):
    """Append, attention and read back over several steps, captured once over static buffers and replayed with eager work
    between, against the same calls made one by one."""
    rng = np.random.default_rng(12)
    batch, start = 5, np.array([1, 15, 16, 40, 200], dtype=np.int32)
    tables, blocks = _tables(rng, start + 8)
    width = tables.shape[1]
    pool = _up(_filled(rng, blocks, 3), device)
    eager = pool.clone()
    capacity = _hip.plan_capacity(batch, width)
    fields = _hip.load().pc_attn_plan_record_ints()
    plan = torch.zeros((capacity, fields), dtype=torch.int32, device=device)
    lens = torch.zeros(batch, dtype=torch.int32, device=device)
    slots = torch.full((batch,), -1, dtype=torch.int64, device=device)
    query, key, value = (torch.zeros((batch, n, 64), dtype=torch.float16, device=device) for n in (32, 4, 4))
    workspace = torch.zeros(_hip.workspace_bytes(batch, width), dtype=torch.uint8, device=device)

    def step():
        out = torch.zeros_like(query)
        back = torch.zeros((2, 1, batch, 4, 64), dtype=torch.float16, device=device)
        _hip.planned_decode_attention_q4(out, query, pool, 3, lens, plan, width, workspace, new_key=key, new_value=value)
        _hip.kv_read_q4(back[0], back[1], pool, 3, slots)
        return out, back

    graph, (out, back) = capture_graph(step, device)
    for turn in range(6):
        lengths = start + 1 + turn
        host = np.zeros((capacity, fields), dtype=np.int32)
        _hip.decode_plan_into(lengths, tables, host)
        plan.copy_(torch.from_numpy(host))
        lens.copy_(torch.from_numpy(lengths))
        at = np.array([tables[b, (n - 1) // 16] * 16 + (n - 1) % 16 for b, n in enumerate(lengths)], dtype=np.int64)
        slots.copy_(torch.from_numpy(at))
        for t in (query, key, value):
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape)).astype(np.float16)))
        graph.replay()
        torch.cuda.synchronize()
        expected = _attend(device, eager, 3, query, tables, lengths, (key, value))
        assert torch.equal(out.view(torch.int16), expected.view(torch.int16))
        assert torch.equal(pool, eager)
        read = torch.zeros_like(back)
        _hip.kv_read_q4(read[0], read[1], eager, 3, slots)
        assert torch.equal(back.view(torch.int16), read.view(torch.int16))
    _hip.check_attention_faults(workspace, "test")


def test_offsets_past_32_bits(device):
    """A pool of over 4 GiB: blocks at its end, in its last layer."""
    blocks = 46000  # 22 * 46000 * 4608 bytes
    pool = _hip.empty_q4_pool(blocks, device)
    pool[21].zero_()
    rng = np.random.default_rng(13)
    length = 100
    table = np.array([[blocks - 1 - 3 * i for i in range(7)]], dtype=np.int32)
    slots = np.array([table[0, p // 16] * 16 + p % 16 for p in range(length)], dtype=np.int64)
    key, value = _rows(rng, 1, length), _rows(rng, 1, length)
    _hip.kv_append_q4(pool, 21, _up(key, device), _up(value, device), _up(slots, device))
    last = pool[21].cpu().numpy()
    expected = np.zeros((22, blocks, 4, ref.UNIT), dtype=np.uint8)[21:]
    ref.write(expected, 0, key, value, slots)
    assert (last == expected[0]).all()
    query = _up(rng.standard_normal((1, 32, 64)).astype(np.float16), device)
    out = _attend(device, pool, 21, query, table, [length])
    _check_rows(out, query, last, table, [length])
    back = torch.zeros((2, 1, length, 4, 64), dtype=torch.float16, device=device)
    _hip.kv_read_q4(back[0], back[1], pool, 21, _up(slots, device))
    for kind in range(2):
        _assert_read(back[kind, 0].cpu().numpy(), ref.rows(last, kind, slots))


def test_nothing_to_do(device):
    """No tokens, no sequences, sequences that are all empty: the pool and the outputs stay as they were."""
    pool = torch.randint(0, 256, (22, 4, 4, ref.UNIT), dtype=torch.uint8, device=device)
    before = pool.clone()
    rows = [torch.empty((3, 0, 4, 64), dtype=torch.float16, device=device) for _ in range(2)]
    slots = torch.empty(0, dtype=torch.int64, device=device)
    _hip.kv_append_q4(pool, 0, *rows, slots)
    _hip.kv_read_q4(*rows, pool, 0, slots)
    for lengths in ([], [0], [0, 0, 0]):
        n = len(lengths)
        lens, tables = torch.zeros(n, dtype=torch.int32, device=device), torch.zeros((n, 2), dtype=torch.int32, device=device)
        query = torch.zeros((n, 32, 64), dtype=torch.float16, device=device)
        out = torch.full_like(query, 3.0)
        workspace = torch.zeros(_hip.workspace_bytes(n, 2), dtype=torch.uint8, device=device)
        _hip.paged_decode_attention_q4(out, query, pool, 1, tables, lens, workspace=workspace)
        new = torch.ones((n, 4, 64), dtype=torch.float16, device=device)
        plan = _up(_hip.decode_plan(np.zeros(n, dtype=np.int32), np.zeros((n, 2), dtype=np.int32)), device)
        _hip.planned_decode_attention_q4(out, query, pool, 1, lens, plan, 2, workspace, new_key=new, new_value=new)
        torch.cuda.synchronize()
        assert (out == 3.0).all() and not workspace.any()
    assert torch.equal(pool, before)


def test_another_stream(device):
    rng = np.random.default_rng(14)
    lengths = [600, 31]
    tables, blocks = _tables(rng, lengths)
    pool = _filled(rng, blocks, 0)
    on = _up(pool, device)
    query = _up(rng.standard_normal((2, 32, 64)).astype(np.float16), device)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out = torch.full_like(query, 3.0)
        lens = np.array(lengths, dtype=np.int32)
        workspace = _hip.paged_decode_attention_q4(out, query, on, 0, _up(tables, device), _up(lens, device))
    stream.synchronize()
    _hip.check_attention_faults(workspace, "test")
    _check_rows(out, query, pool[0], tables, lengths)
