"""Calls whose work takes 2^32 threads or more, which a launch counts modulo 2^32 without an error."""

from __future__ import annotations

import ctypes

import pytest
import torch

from pagedcore_amd import _hip


def test_refused():
    lib = _hip.load()
    buffer = ctypes.create_string_buffer(1 << 12)
    at = (ctypes.addressof(buffer) + 255) // 256 * 256
    assert lib.pc_add_rms_norm(at, at, None, at, 1 << 24, 8, 1e-5, None) == 1 and b"too large" in lib.pc_last_error()
    assert lib.pc_silu_mul(at, at, 1 << 32, 8, None) == 1 and b"too large" in lib.pc_last_error()
    tokens = (1 << 32) // 192 + 1
    assert lib.pc_rope_kv_append(at, None, None, at, 2560, at, at, 8, None, 0, 0, None, tokens, None) == 1 and b"too large" in lib.pc_last_error()


@pytest.mark.gpu
def test_fp16_append_of_rows_at_odd_addresses(device):
    """2^23 tokens and some, a word a thread; a token stride of 0, and all but a few slots outside the pool."""
    tokens = (1 << 23) + 21
    wide = torch.randn(2, 257, dtype=torch.float16, device=device)
    key, value = (row[1:].view(1, 1, 4, 64).expand(1, tokens, 4, 64) for row in wide)
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=device)
    at = torch.tensor([0, 5, (1 << 22) - 1, 1 << 22, (1 << 23) - 1, 1 << 23, tokens - 1], device=device)
    slots[at] = torch.arange(20, 27, device=device)
    pool = torch.full((22, 2, 2, 16, 4, 64), 7.0, dtype=torch.float16, device=device)
    expected = pool.clone()
    expected.view(22, 2, 32, 4, 64)[3, :, 20:27] = wide[:, 1:].reshape(2, 1, 4, 64)
    _hip.kv_append(pool, 3, key, value, slots)
    assert torch.equal(pool, expected)
