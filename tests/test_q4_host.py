"""The 4-bit KV pool without a GPU: the oracle's format against the definition, what the binding and the library refuse, the
allocator's bookkeeping over a 4-bit pool."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import q4_reference as ref
from pagedcore_amd import _hip
from pagedcore_amd.config import PagedCoreConfig
from pagedcore_amd.engine_types import KVReservation, RequestId
from pagedcore_amd.kv_cache import HipQ4Writer, KVAllocator, allocate_kv_pool
from tests.test_fp8_devices import OnGpu, calls  # noqa: F401  (the fixture)

# --- the format --------------------------------------------------------------------------


def test_every_value_has_its_own_bits():
    for kind, place in enumerate((ref.key_place, ref.value_place)):
        taken = np.zeros((ref.UNIT, 8), dtype=int)
        for t in range(16):
            for d in range(64):
                byte, bit = place(t, d)
                taken[byte, bit : bit + 4] += 1
        assert (taken[512 * kind : 512 * kind + 512] == 1).all() and taken.sum() == 4096
    pairs = sorted(ref.pair_place(kind, t) for kind in range(2) for t in range(16))
    assert pairs == list(range(1024, 1152, 4))


def test_bytes_belong_to_one_slot():
    """A slot is written without reading its neighbours: no byte holds bits of two."""
    for place in (ref.key_place, ref.value_place):
        owners = {}
        for t in range(16):
            for d in range(64):
                assert owners.setdefault(place(t, d)[0], t) == t


def test_quantize_by_hand():
    x = np.zeros((1, 64), dtype=np.float16)
    x[0, :16] = np.arange(16)
    n, lo, s = ref.quantize(x)
    assert lo[0] == 0 and s[0] == 1 and list(n[0, :16]) == list(range(16)) and (n[0, 16:] == 0).all()
    x[0] = 3.0
    n, lo, s = ref.quantize(x)
    assert lo[0] == 3 and s[0] == 0 and (n == 0).all()
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = -1.0, 29.0, 0.0, 2.0  # steps of 2: 0.5 and 1.5 levels up are ties
    n, lo, s = ref.quantize(x)
    assert lo[0] == -1 and s[0] == 2 and list(n[0, :4]) == [0, 15, 0, 2]
    x[0, 0], x[0, 1:] = 0.0, 1.0  # fifteen steps reach the largest value: s is rounded up
    n, lo, s = ref.quantize(x)
    assert float(s[0]) * 15 >= 1 > float(np.nextafter(s[0], np.float16(0))) * 15 and n[0, 1] == 15
    for bad in (np.nan, np.inf, -np.inf):
        x[0, 7] = bad
        n, lo, s = ref.quantize(x)
        assert np.isnan(lo[0]) and s[0] == 0 and (n == 0).all()


def test_written_rows_read_back_within_half_a_step():
    rng = np.random.default_rng(0)
    pool = rng.integers(0, 256, (22, 3, 4, ref.UNIT), dtype=np.uint8)
    key, value = (rng.standard_normal((2, 20, 4, 64)).astype(np.float16) for _ in range(2))
    slots = rng.permutation(48)[:20]
    ref.write(pool, 5, key, value, slots)
    for kind, rows in enumerate((key, value)):
        for layer in range(2):
            got = ref.rows(pool[5 + layer], kind, slots)
            _, _, s = ref.quantize(rows[layer])
            assert (np.abs(got - rows[layer]) <= s.astype(np.float64)[..., None] / 2).all()


# --- the binding -------------------------------------------------------------------------


def _on(shape, dtype=torch.float16, gpu=0):
    return OnGpu(torch.zeros(shape, dtype=dtype), gpu)


def _call(**kw):
    pool, key, slots = _on((22, 3, 4, 1152), torch.uint8), _on((2, 5, 4, 64)), _on((5,), torch.int64)
    return kw.get("pool", pool), kw.get("key", key), kw.get("value", _on((2, 5, 4, 64))), kw.get("slots", slots), kw.get("begin", 0)


@pytest.mark.parametrize("change,match", [
    ({"pool": _on((22, 3, 4, 1152))}, "uint8"),
    ({"pool": _on((22, 2, 3, 16, 4, 64))}, "uint8"),
    ({"pool": _on((21, 3, 4, 1152), torch.uint8)}, "uint8"),
    ({"pool": _on((22, 0, 4, 1152), torch.uint8)}, "uint8"),
    ({"pool": _on((22, 3, 4, 1151), torch.uint8)}, "uint8"),
    ({"pool": OnGpu(torch.zeros((22, 3, 4, 2304), dtype=torch.uint8)[..., ::2], 0)}, "contiguous uint8"),
    ({"pool": torch.zeros((22, 3, 4, 1152), dtype=torch.uint8)}, "not the current GPU"),
    ({"key": _on((2, 5, 4, 32))}, "share"),
    ({"key": _on((2, 5, 8, 64))}, "share"),
    ({"key": _on((5, 4, 64))}, "share"),
    ({"value": _on((2, 4, 4, 64))}, "share"),
    ({"begin": 21}, "within 22"),
    ({"begin": -1}, "within 22"),
    ({"key": _on((0, 5, 4, 64)), "value": _on((0, 5, 4, 64))}, "within 22"),
    ({"key": _on((2, 5, 4, 64), torch.float32)}, "float16"),
    ({"value": _on((2, 5, 4, 64), torch.bfloat16)}, "float16"),
    ({"key": _on((2, 5, 4, 64), gpu=1)}, "GPU 0"),
    ({"slots": _on((5,), torch.int32)}, "slot_mapping"),
    ({"slots": _on((4,), torch.int64)}, "slot_mapping"),
    ({"slots": _on((5, 1), torch.int64)}, "slot_mapping"),
    ({"slots": OnGpu(torch.zeros(10, dtype=torch.int64)[::2], 0)}, "slot_mapping"),
    ({"slots": _on((5,), torch.int64, gpu=1)}, "slot_mapping"),
])
def test_rows_refused(calls, change, match):  # noqa: F811
    pool, key, value, slots, begin = _call(**change)
    with pytest.raises(_hip.HipExtensionError, match=match):
        _hip.kv_append_q4(pool, begin, key, value, slots)
    with pytest.raises(_hip.HipExtensionError, match=match):
        _hip.kv_read_q4(key, value, pool, begin, slots)
    assert calls == []


def test_rows_to_read_into_must_be_whole(calls):  # noqa: F811
    pool, key, value, slots, _ = _call()
    with pytest.raises(_hip.HipExtensionError, match="contiguous"):
        _hip.kv_read_q4(OnGpu(torch.zeros((2, 5, 64, 4), dtype=torch.float16).transpose(2, 3), 0), value, pool, 0, slots)
    assert calls == []


@pytest.mark.parametrize("rows", [
    torch.zeros((1, 5, 4, 64), dtype=torch.float16).expand(2, 5, 4, 64),
    torch.zeros((2, 1, 4, 64), dtype=torch.float16).expand(2, 5, 4, 64),
    torch.zeros(2000, dtype=torch.float16).as_strided((2, 5, 4, 64), (400, 128, 64, 1)),
])
def test_rows_to_read_into_must_not_overlap(calls, rows):  # noqa: F811
    pool, _, value, slots, _ = _call()
    for pair in ((OnGpu(rows, 0), value), (value, OnGpu(rows, 0))):
        with pytest.raises(_hip.HipExtensionError, match="overlap"):
            _hip.kv_read_q4(*pair, pool, 0, slots)
    assert calls == []
    single = OnGpu(torch.zeros((1, 1, 4, 64), dtype=torch.float16).as_strided((1, 1, 4, 64), (0, 0, 64, 1)), 0)
    _hip.kv_read_q4(single, single, pool, 0, _on((1,), torch.int64))  # one row: its strides are of no account
    _hip.kv_append_q4(pool, 0, OnGpu(rows, 0), value, slots)  # what is only read may
    assert [name for name, *_ in calls] == ["pc_kv_read_q4", "pc_kv_append_q4"]


def test_calls_go_to_the_pools_gpu(calls):  # noqa: F811
    for gpu in (0, 2):
        on = lambda shape, dtype=torch.float16: _on(shape, dtype, gpu)  # noqa: E731
        pool, key, value, slots = on((22, 3, 4, 1152), torch.uint8), on((1, 2, 4, 64)), on((1, 2, 4, 64)), on((2,), torch.int64)
        _hip.kv_append_q4(pool, 3, key, value, slots)
        _hip.kv_read_q4(key, value, pool, 3, slots)
    assert calls == [(name, gpu, 7000 + gpu) for gpu in (0, 2) for name in ("pc_kv_append_q4", "pc_kv_read_q4")]


def test_attention_refused(monkeypatch):
    library = _hip.load()
    launched = []

    class Library:
        def __getattr__(self, name):
            if name in ("pc_paged_decode_attn_q4", "pc_kv_append_paged_decode_attn_q4"):
                return lambda *args: launched.append(name) or 0
            return getattr(library, name)

    monkeypatch.setattr(_hip, "load", lambda: Library())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_hip, "_raw_stream", lambda index: 7)
    good = {
        "out": _on((3, 32, 64)), "query": _on((3, 32, 1, 64)), "pool": _on((22, 3, 4, 1152), torch.uint8), "layer": 0,
        "context_lens": _on((3,), torch.int32), "plan": _on((8, 296), torch.int32), "max_blocks": 2,
        "workspace": _on((_hip.workspace_bytes(3, 2),), torch.uint8),
    }
    _hip.planned_decode_attention_q4(**good)
    _hip.planned_decode_attention_q4(**good, new_key=_on((3, 4, 64)), new_value=_on((3, 4, 64)))
    assert launched == ["pc_paged_decode_attn_q4", "pc_kv_append_paged_decode_attn_q4"]
    for change, match in (
        ({"out": _on((3, 32, 63))}, "out"),
        ({"out": _on((2, 32, 64))}, "out"),
        ({"query": _on((3, 32, 64), torch.float32)}, "query"),
        ({"query": OnGpu(torch.zeros((3, 64, 64), dtype=torch.float16)[:, ::2], 0)}, "query"),
        ({"query": _on((3, 32, 64), gpu=1)}, "query"),
        ({"pool": _on((22, 2, 3, 16, 4, 64))}, "uint8"),
        ({"context_lens": _on((3,), torch.int64)}, "context_lens"),
        ({"context_lens": _on((3, 1), torch.int32)}, "context_lens"),
        ({"plan": _on((8, 295), torch.int32)}, "plan"),
        ({"plan": _on((8, 296), torch.int64)}, "plan"),
        ({"max_blocks": 0}, "shape"),
        ({"max_blocks": 65537}, "shape"),
        ({"workspace": _on((_hip.workspace_bytes(3, 2) - 1,), torch.uint8)}, "workspace"),
        ({"new_key": _on((3, 4, 64))}, "together"),
        ({"new_value": _on((3, 4, 64))}, "together"),
        ({"new_key": _on((3, 4, 32)), "new_value": _on((3, 4, 64))}, "new_key"),
        ({"new_key": _on((3, 4, 64)), "new_value": _on((3, 4, 64), torch.float32)}, "new_value"),
    ):
        with pytest.raises(_hip.HipExtensionError, match=match):
            _hip.planned_decode_attention_q4(**{**good, **change})
    assert len(launched) == 2


def test_the_fp16_calls_look_at_no_other_type():
    """Their rows are 16-bit words: what they took before there were 4-bit pools, they still take."""
    for dtype in (torch.float16, torch.int16, torch.bfloat16):
        _hip._check_fp16_pool(torch.zeros((22, 2, 1, 16, 4, 64), dtype=dtype))
    _hip._check_fp16_pool(None)


def test_the_fp16_calls_refuse_a_4_bit_pool():
    pool = torch.zeros((22, 3, 4, 1152), dtype=torch.uint8)
    rows = torch.zeros((1, 2, 4, 64), dtype=torch.float16)
    slots = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(_hip.HipExtensionError, match="float16"):
        _hip.kv_append(pool, 0, rows, rows, slots)
    with pytest.raises(_hip.HipExtensionError, match="float16"):
        _hip.rope_kv_append(rows, torch.zeros((2, 2560), dtype=torch.float16), slots, rows, pool=pool, slot_mapping=slots)
    lens, plan = torch.zeros(2, dtype=torch.int32), torch.zeros((8, 296), dtype=torch.int32)
    with pytest.raises(_hip.HipExtensionError, match="float16"):
        _hip.planned_decode_attention(rows, rows, pool, 0, lens, plan, 1, torch.zeros(1 << 22, dtype=torch.uint8))


# --- the library's own checks (no launch: every call below is refused, or has nothing to do) ---


def test_library_refusals():
    lib = _hip.load()
    buffer = ctypes.create_string_buffer(1 << 16)
    at = (ctypes.addressof(buffer) + 255) // 256 * 256

    def append(**kw):
        return lib.pc_kv_append_q4(
            kw.get("pool", at), kw.get("blocks", 3), kw.get("begin", 0), kw.get("layers", 1), kw.get("key", at), 256, 256,
            kw.get("value", at), 256, 256, kw.get("slots", at), kw.get("tokens", 1), None,
        )

    def read(**kw):
        return lib.pc_kv_read_q4(
            kw.get("key", at), 256, 256, kw.get("value", at), 256, 256, kw.get("pool", at), kw.get("blocks", 3), kw.get("begin", 0),
            kw.get("layers", 1), kw.get("slots", at), kw.get("tokens", 1), None,
        )

    for call in (append, read):
        assert call(tokens=0) == 0 and call(tokens=0, key=None, value=None, slots=None) == 0  # as empty tensors' pointers are
        for change, text in (
            ({"pool": None}, b"null"), ({"key": None}, b"null"), ({"value": None}, b"null"), ({"slots": None}, b"null"),
            ({"blocks": 0}, b"num_blocks"), ({"blocks": (1 << 26) + 1}, b"num_blocks"), ({"begin": -1}, b"layers"),
            ({"begin": 21, "layers": 2}, b"layers"), ({"begin": 2147483647, "layers": 22}, b"layers"), ({"layers": 0}, b"layers"),
            ({"tokens": -1}, b"negative"), ({"tokens": 1 << 29}, b"too many"), ({"pool": at + 64}, b"128-byte"),
            ({"key": at + 1}, b"2-byte"), ({"slots": at + 4}, b"8-byte"),
        ):
            assert call(**change) == 1 and text in lib.pc_last_error(), (change, lib.pc_last_error())

    def attend(fused, **kw):
        args = [kw.get("out", at), kw.get("query", at), kw.get("pool", at), kw.get("blocks", 3), kw.get("layer", 0), kw.get("lens", at),
                kw.get("batch", 1), kw.get("width", 1), kw.get("plan", at), kw.get("rows", 8)]
        if fused:
            return lib.pc_kv_append_paged_decode_attn_q4(*args, kw.get("key", at), kw.get("value", at), kw.get("workspace", at), None)
        return lib.pc_paged_decode_attn_q4(*args, kw.get("workspace", at), None)

    for fused in (False, True):
        assert attend(fused, rows=0) == 0 and attend(fused, batch=0) == 0
        assert attend(fused, rows=0, plan=None) == 0  # nothing but empty sequences
        assert attend(fused, batch=0, rows=0, out=None, query=None, lens=None, plan=None, key=None, value=None) == 0
        for change, text in (
            ({"out": None}, b"null"), ({"plan": None}, b"null"), ({"workspace": None}, b"workspace"), ({"blocks": 0}, b"num_blocks"),
            ({"blocks": (1 << 26) + 1}, b"num_blocks"), ({"layer": 22}, b"layer"), ({"layer": -1}, b"layer"), ({"batch": -1}, b"batch"),
            ({"width": 0}, b"max_blocks"), ({"query": at + 8}, b"aligned"), ({"pool": at + 16}, b"aligned"),
            ({"workspace": at + 128}, b"aligned"), ({"rows": -1}, b"num_records"), ({"rows": 1 << 20}, b"num_records"),
        ):
            assert attend(fused, **change) == 1 and text in lib.pc_last_error(), (change, lib.pc_last_error())
    assert attend(True, key=None) == 1 and attend(True, value=at + 2) == 1


# --- the allocator -----------------------------------------------------------------------


def test_pool_sizes_and_refusals(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (16 * 2**30, 16 * 2**30))
    monkeypatch.setattr(_hip, "empty_q4_pool", lambda blocks, device: torch.empty((22, blocks, 4, 1152), dtype=torch.uint8, device="meta"))
    pool = allocate_kv_pool(PagedCoreConfig(kv_pool_mib=8192), bits=4)
    assert pool.shape[1] == 8192 * 2**20 // (99 * 1024) and pool.shape[1] > 3.5 * 23831
    for bits in (8, 0, 4.0, True, "4"):
        with pytest.raises(ValueError, match="16 or 4 bits"):
            allocate_kv_pool(PagedCoreConfig(), bits=bits)


def test_bookkeeping_over_a_cpu_pool():
    pool = torch.zeros((22, 6, 4, 1152), dtype=torch.uint8)
    allocator = KVAllocator(pool)
    assert allocator.quantized and allocator.total_blocks == 6
    request = RequestId("a")
    allocator.create(KVReservation(request, 3))
    assert allocator.capacity().total_blocks == 6 and allocator.capacity().reserved_blocks == 3
    rows = torch.zeros((22, 4, 4, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CPU"):
        allocator.append(request, rows, rows)
    assert allocator.cached_length(request) == 0 and allocator.capacity().free_blocks == 6

    class Counted(HipQ4Writer):
        def __init__(self):
            self.calls = []

        def append(self, pool, layer_begin, key, value, slots):
            self.calls.append((layer_begin, tuple(key.shape), list(slots)))

    writer = Counted()
    allocator = KVAllocator(pool, kv_writer=writer)
    allocator.create(KVReservation(request, 3))
    allocator.append(request, rows.expand(22, 4, 4, 64), rows)
    assert writer.calls == [(0, (22, 4, 4, 64), [0, 1, 2, 3])] and allocator.cached_length(request) == 4
    for read in (lambda: allocator.read_block(request, 0), lambda: list(allocator.iter_layer_blocks(request, layer_index=0))):
        with pytest.raises(RuntimeError, match="4-bit pool"):
            read()
    allocator.release_all(request)
    assert allocator.capacity().free_blocks == 6


@pytest.mark.parametrize("pool", [
    torch.zeros((22, 6, 4, 1151), dtype=torch.uint8), torch.zeros((21, 6, 4, 1152), dtype=torch.uint8),
    torch.zeros((22, 0, 4, 1152), dtype=torch.uint8), torch.zeros((22, 6, 4, 1152), dtype=torch.int8),
    torch.zeros((22, 6, 4, 2304), dtype=torch.uint8)[..., ::2], torch.zeros((22, 2, 6, 16, 4, 64), dtype=torch.uint8),
])
def test_other_pools_are_refused(pool):
    with pytest.raises(ValueError, match="KV pool must be"):
        KVAllocator(pool)
