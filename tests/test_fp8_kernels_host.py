"""Which kernels the 8-bit projections take, asked of the library's own choice, without a GPU."""

from __future__ import annotations

import pytest

from pagedcore_amd import _hip

PARTIALS, HALF, SWIGLU, SWIGLU_FP8, ROPE = 0, 1, 2, 4, 5
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
