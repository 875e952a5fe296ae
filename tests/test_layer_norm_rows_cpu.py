"""The C entries of layer norm of 16-bit rows, as far as they go without a device."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from csn_b200 import _build, _lib
    _build.build()
    return _lib.load()


null = ctypes.c_void_p(0)


@pytest.mark.parametrize("C", [1, 64, 771, 8192, 20000])
@pytest.mark.parametrize("dtype,weight_dtype", [(1, 1), (1, 0), (2, 2)])
def test_backward_without_rows_launches_nothing(lib, C, dtype, weight_dtype):
    """No rows and no weight, which is not wanted then: there is nothing to read, and without gradients nothing to write."""
    assert lib.csn_layer_norm_rows_bwd(null, C, null, C, null, null, null, null, null, null, 0, C, dtype, weight_dtype, null, 0, null) == 0
