"""What the binding of the 4-bit KV pool's calls takes and refuses, without a GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from pagedcore_amd import _hip
from tests.test_fp8_devices import OnGpu, calls  # noqa: F401  (the fixture)


def _pool():
    return OnGpu(torch.zeros((22, 3, 4, 1152), dtype=torch.uint8), 0)


def _view(base, offset, layers, tokens, layer_stride, token_stride):
    return OnGpu(base.as_strided((layers, tokens, 4, 64), (layer_stride, token_stride, 64, 1), offset), 0)


# (offset, layer stride, token stride) of K and of V, in elements of one buffer; layers, tokens; whether a row meets another
SHARED = [
    ((0, 1280, 256), (0, 1280, 256), 2, 5, True),  # one tensor for both
    ((0, 1280, 256), (255, 1280, 256), 2, 5, True),
    ((0, 1280, 256), (2 * 1280 - 1, 1280, 256), 2, 5, True),  # the last row's last element
    ((0, 1280, 256), (2 * 1280, 1280, 256), 2, 5, False),  # one behind the other
    ((2560, 1280, 256), (0, 1280, 256), 2, 5, False),
    ((0, 2560, 512), (256, 2560, 512), 2, 5, False),  # K and V of a token side by side
    ((0, 2560, 512), (255, 2560, 512), 2, 5, True),
    ((0, 2560, 512), (257, 2560, 512), 2, 5, True),
    ((256, 2560, 512), (0, 2560, 512), 2, 5, False),
    ((0, 2560, 256), (1280, 2560, 256), 2, 5, False),  # of a layer
    ((0, 2560, 256), (1279, 2560, 256), 2, 5, True),
    ((0, 2560, 256), (1281, 2560, 256), 2, 5, True),
    ((0, 256, 512), (5120, 256, 512), 2, 5, False),  # tokens outside, layers inside
    ((0, 256, 1024), (512, 256, 1024), 2, 5, False),
    ((0, 256, 1024), (256, 256, 1024), 2, 5, True),  # K's second layer is V's first
    ((0, 1280, 256), (2560, 2048, 512), 2, 4, False),  # strides of their own
    ((0, 2048, 512), (256, 4096, 1024), 2, 4, False),
    ((0, 2048, 512), (256, 4096, 1025), 2, 4, True),
    ((0, 0, 512), (256, 0, 512), 1, 7, False),  # one layer: its stride is of no account
    ((0, 0, 512), (512, 0, 512), 1, 7, True),
    ((0, 512, 0), (256, 512, 0), 3, 1, False),
    ((0, 512, 0), (512, 512, 0), 3, 1, True),
    ((0, 0, 0), (256, 0, 0), 1, 1, False),
    ((0, 0, 0), (255, 0, 0), 1, 1, True),
    ((0, 0, 0), (0, 0, 0), 1, 0, False),  # no rows at all
]


@pytest.mark.parametrize("key,value,layers,tokens,meet", SHARED)
def test_key_and_value_must_not_share_rows(calls, key, value, layers, tokens, meet):  # noqa: F811
    base = torch.zeros(20000, dtype=torch.float16)
    elements = lambda at: {at[0] + layer * at[1] + t * at[2] + i for layer in range(layers) for t in range(tokens) for i in range(256)}  # noqa: E731
    assert bool(elements(key) & elements(value)) == meet
    rows = [_view(base, offset, layers, tokens, *strides) for offset, *strides in (key, value)]
    slots = OnGpu(torch.zeros(tokens, dtype=torch.int64), 0)
    if meet:
        with pytest.raises(_hip.HipExtensionError, match="overlap"):
            _hip.kv_read_q4(*rows, _pool(), 0, slots)
        assert calls == []
    else:
        _hip.kv_read_q4(*rows, _pool(), 0, slots)
        assert [name for name, *_ in calls] == ["pc_kv_read_q4"]
    _hip.kv_append_q4(_pool(), 0, *rows, slots)  # what is only read may overlap
    assert calls[-1][0] == "pc_kv_append_q4"


def test_rows_that_meet_against_every_element():
    rng = np.random.default_rng(0)
    seen = [0, 0]
    for _ in range(4000):
        layers, tokens = (int(n) for n in rng.integers(1, 5, 2))
        places = []
        for _ in range(2):
            inner = int(rng.integers(256, 900))
            strides = (inner, 256 + inner * (layers - 1)) if rng.random() < 0.3 else (256 + inner * (tokens - 1) + int(rng.integers(0, 700)), inner)
            places.append(strides)
        if rng.random() < 0.5:
            places[1] = places[0]
        distance = int(rng.integers(-3000, 3000))
        at = [np.add.outer(np.arange(layers) * s[0], np.arange(tokens) * s[1]).reshape(-1) for s in places]
        meet = bool((abs(at[0][:, None] - (at[1] + distance)) < 256).any())
        seen[meet] += 1
        assert _hip._rows_meet(distance, places[0], places[1], layers, tokens) == meet
    assert min(seen) > 500


def test_attention_rows_are_told_by_their_whole_shape(calls, monkeypatch):  # noqa: F811
    """Rows of as many elements in another order are refused, not read as [batch, heads, 64]; dimensions of 1 between are taken."""
    on = lambda shape, dtype=torch.float16: OnGpu(torch.zeros(shape, dtype=dtype), 0)  # noqa: E731
    stand_in = _hip.load()

    class Library:
        def __getattr__(self, name):
            return (lambda *args: 1 << 20) if name == "pc_attn_workspace_bytes" else getattr(stand_in, name)

    monkeypatch.setattr(_hip, "load", lambda: Library())
    good = {
        "out": on((3, 32, 64)), "query": on((3, 32, 64)), "pool": _pool(), "layer": 0, "context_lens": on((3,), torch.int32),
        "plan": on((8, 296), torch.int32), "max_blocks": 2, "workspace": on((1 << 20,), torch.uint8), "new_key": on((3, 4, 64)),
        "new_value": on((3, 4, 64)),
    }
    for name, heads in (("out", 32), ("query", 32), ("new_key", 4), ("new_value", 4)):
        for shape in ((3, 64, heads), (3, heads * 64), (3, heads // 2, 128), (3, 2, heads // 2, 64), (3 * heads, 64), (heads, 3, 64), (3, 64, heads, 1), (3 * heads * 64,)):
            with pytest.raises(_hip.HipExtensionError, match=name):
                _hip.planned_decode_attention_q4(**{**good, name: on(shape)})
    assert calls == []
    for name, heads in (("out", 32), ("query", 32), ("new_key", 4), ("new_value", 4)):
        for shape in ((3, heads, 1, 64), (3, 1, heads, 64), (3, 1, heads, 1, 64)):
            _hip.planned_decode_attention_q4(**{**good, name: on(shape)})
    assert [name for name, *_ in calls] == ["pc_kv_append_paged_decode_attn_q4"] * 12


def test_the_fp16_calls_take_a_pool_as_bytes(calls):  # noqa: F811
    """The fp16 pool as uint8 [22, 2, blocks, 16, 4, 128] went through its calls before there were 4-bit pools, and does now."""
    pool = torch.zeros((22, 2, 3, 16, 4, 64), dtype=torch.float16).view(torch.uint8)
    rows, slots = torch.zeros((1, 2, 4, 64), dtype=torch.float16), torch.zeros(2, dtype=torch.int64)
    _hip.kv_append(pool, 0, rows, rows, slots)
    _hip.rope_kv_append(rows, torch.zeros((2, 2560), dtype=torch.float16), slots, rows, pool=pool, slot_mapping=slots)
    assert [name for name, *_ in calls] == ["pc_kv_append", "pc_rope_kv_append"]


def test_plans_of_more_rows_than_a_launch_has_threads_for():
    """A plan padded to a capacity of 2^23 rows and more (of 512 threads each; 2^24 of the fp16 kernel's 256) is refused."""
    lib = _hip.load()
    buffer = ctypes.create_string_buffer(1 << 12)
    at = (ctypes.addressof(buffer) + 255) // 256 * 256
    assert _hip.plan_capacity(1 << 20, 1 << 16) > 1 << 30
    shape = (at, at, at, 3, 0, at, 1 << 20, 1 << 16, at)
    for rows in (1 << 23, (1 << 23) + 1, 1 << 29):
        assert lib.pc_paged_decode_attn_q4(*shape, rows, at, None) == 1 and b"8388600" in lib.pc_last_error()
        assert lib.pc_kv_append_paged_decode_attn_q4(*shape, rows, at, at, at, None) == 1 and b"8388600" in lib.pc_last_error()
        assert lib.pc_paged_decode_attn(*shape, 2 * rows, at, None) == 1 and b"16777208" in lib.pc_last_error()
        assert lib.pc_kv_append_paged_decode_attn(*shape, 2 * rows, at, at, at, None) == 1 and b"16777208" in lib.pc_last_error()
