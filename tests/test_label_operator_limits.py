"""Limits of the label-selection operators that the C ABI checks before any launch, so they run without a GPU."""
import ctypes

import pytest

one = ctypes.c_void_p(16)            # never dereferenced: the checks fail first
F32 = 0


@pytest.fixture(scope="module")
def L():
    from semantic_segmentation_amd import _lib
    return _lib.lib


@pytest.mark.parametrize("t", [1e-30, 9.9e-19, 1.1e18, 1e30])
def test_distillation_refuses_temperatures_whose_square_is_no_fp32_number(t, L):
    v = (one, F32, 2, 5, 3, 15, 3, 1)
    assert L.mfl_distillation_forward(*v, one, F32, one, None, None, 2, t, one, one, None, 0, None) == -1
    assert L.mfl_distillation_backward(*v, one, F32, one, None, None, 2, t, one, one, one, 15, 3, 1, None) == -1
