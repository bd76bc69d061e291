"""Which kernels the 8-bit projections take, asked of the library's own choice, without a GPU."""

from __future__ import annotations

import pytest

from pagedcore_amd import _hip
from pagedcore_amd import decoder as dec
from tests import fp8_sizes
from tests.fp8_sizes import HALF, PARTIALS, ROPE, SWIGLU, SWIGLU_FP8

FORMS = [(PARTIALS, 0), (PARTIALS, 1), (HALF, 0), (HALF, 1), (SWIGLU, 0), (SWIGLU, 1), (SWIGLU_FP8, 0), (ROPE, 0), (ROPE, 1)]


def kernel(form, half_x, m, n, k, splits=1):
    return _hip.load().pc_gemm_fp8_kernel(m, n, k, splits, form, half_x)


@pytest.mark.parametrize("form,half_x", FORMS)
def test_a_call_has_one_of_its_forms_kernels(form, half_x):
    count = _hip.load().pc_gemm_fp8_kernels(form, half_x)
    assert 0 < count < 32
    for m in (1, 2, 17, 64, 100, 128, 129, 333, 2048, 65536):
        taken = kernel(form, half_x, m, 2560, 2048)
        assert taken == -1 if m > 128 and (half_x or form == PARTIALS) else 0 <= taken < count


@pytest.mark.parametrize("form,half_x", [(3, 0), (6, 0), (-1, 0), (SWIGLU_FP8, 1)])
def test_no_such_form(form, half_x):
    assert _hip.load().pc_gemm_fp8_kernels(form, half_x) == 0
    assert kernel(form, half_x, 8, 2560, 2048) == -1


@pytest.mark.parametrize("form,m,n,k,splits", [
    (HALF, 0, 64, 128, 1), (HALF, 65537, 64, 128, 1), (HALF, 8, 0, 128, 1), (HALF, 8, 6, 128, 1), (HALF, 8, 64, 24, 1), (HALF, 8, 64, 0, 1),
    (HALF, 8, 64, 128, 2), (SWIGLU, 8, 4, 128, 1), (SWIGLU_FP8, 8, 48, 128, 1), (PARTIALS, 129, 64, 128, 1), (PARTIALS, 8, 64, 128, 2),
    (PARTIALS, 8, 64, 128, 0), (HALF, 65536, 64, 65536, 1), (ROPE, 8, 2048, 128, 1), (ROPE, 8, 2560, (1 << 18) + 16, 1),
])
def test_sizes_that_are_refused_have_no_kernel(form, m, n, k, splits):
    assert kernel(form, 0, m, n, k, splits) == -1


@pytest.mark.parametrize("m", [1, 17, 97, 200, 500, 1000, 2048])
def test_q_k_v_takes_one_kernel_rotated_or_not(m):
    """So that a cache holds the same bytes whichever way the product went into it."""
    assert kernel(HALF, 0, m, 2560, 2048) == kernel(ROPE, 0, m, 2560, 2048)


def _kernels(form, half_x, group):
    return {kernel(form, half_x, *size) for size in fp8_sizes.GROUPS[group].get((form, half_x), [])}


@pytest.mark.parametrize("group", ["RAGGED", "WHOLE"])
@pytest.mark.parametrize("form,half_x", FORMS)
def test_the_tests_sizes_run_every_kernel(form, half_x, group):
    """A change of the choice's constants that takes the sizes off a kernel fails here: other sizes for it are due in
    tests/fp8_sizes.py, or the kernel is one that no call takes."""
    every = set(range(_hip.load().pc_gemm_fp8_kernels(form, half_x)))
    if form == ROPE:
        every -= {5, 6} if not half_x else {3, 4}  # tiles of 24 columns, more quads than threads; eight waves
    assert _kernels(form, half_x, group) == every
    for m, n, k, *_ in fp8_sizes.GROUPS[group][form, half_x]:
        assert (m % 16 and k % 128 and (n % 64 or form == ROPE)) if group == "RAGGED" else m % 16 == n % 64 == k % 128 == 0


def test_the_tests_sizes_run_every_kernel_of_the_model():
    """Of the decoder's calls at 1 to 2048 rows, at its own widths."""
    taken = {}
    for m in range(1, 2049):
        calls = [(ROPE, 0, m, 2560, 2048, 1), (HALF, 0, m, 2560, 2048, 1)]
        if m <= dec.FP8_FUSED_ROWS:
            calls += [(PARTIALS, 1, m, 2048, 2048, dec.FP8_O_PROJ_SPLITS), (PARTIALS, 1, m, 2048, 5632, dec._fp8_down_splits(m))]
        else:
            calls += [(HALF, 0, m, 2048, 2048, 1), (HALF, 0, m, 2048, 5632, 1)]
        calls.append((SWIGLU if m <= dec.FP8_SWIGLU_ROWS else SWIGLU_FP8, 0, m, 11264, 2048, 1))
        for form, half_x, *size in calls:
            taken.setdefault((form, half_x), set()).add(kernel(form, half_x, *size))
    for (form, half_x), kernels in taken.items():
        assert kernels <= _kernels(form, half_x, "MODEL"), (form, half_x)


def test_the_tests_sizes_wrap_every_tile_kernels_scales():
    """Its ring holds the scales of 16 blocks twice: a second fetch behind 2048 columns, the first slot again behind 4096."""
    for form, depths in ((HALF, (2064, 4112, 5632)), (SWIGLU_FP8, (2064, 4112, 5632)), (SWIGLU, (4112,)), (ROPE, (4112,))):
        count = _hip.load().pc_gemm_fp8_kernels(form, 0)
        tiles = set(range(count)) if form == SWIGLU_FP8 else set(range(count - 5, count))
        for depth in depths:
            assert {kernel(form, 0, m, n, k) for m, n, k in fp8_sizes.DEEP[form, 0] if k == depth} == tiles
