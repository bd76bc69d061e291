"""The build's resource check knows the 4-bit pool's kernels whose speed rests on their waves (CPU only)."""

from __future__ import annotations

import os

import pytest

from tests.test_build_guard import _build_module

KERNELS = {"paged_decode_q4_kernel": (4, 8), "kv_append_q4_groups_kernel": (8, 1)}  # waves a SIMD, instances


@pytest.mark.parametrize("kernel", list(KERNELS))
def test_guarded(tmp_path, kernel):
    build = _build_module()
    waves, instances = KERNELS[kernel]
    assert build.GUARDED_KERNELS.get(kernel) == waves
    source = "q4_attention.hip" if "decode" in kernel else "q4_rows.hip"
    text = build.compile_library([os.path.join(build.HERE, name) for name in (source, "pagedcore_hip.hip")], str(tmp_path / "lib.so"))
    assert len(build.check_resource_usage(text, {kernel: waves})) == instances
    with pytest.raises(build.ResourceCheckError, match="waves/SIMD its launch shape assumes"):
        build.check_resource_usage(text, {kernel: waves + 1})
