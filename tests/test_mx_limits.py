"""What the microscaled operators decline, and that they decline it before a launch."""

import ctypes

import pytest
import torch


def _lib():
    import jakal_net_native as jn

    return jn._LIB


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are no memory, should a call not be declined")
def test_products_of_more_tiles_than_a_grid_has_threads_for():
    """A grid has fewer than 2^32 threads: 2^24 tiles of 256 threads, or 2^23 of 512, are one too many."""
    lib, p, many, all_ = _lib(), ctypes.c_void_p(4096), (1 << 31) - 1, ctypes.c_size_t(1 << 62)
    for kind in (0, 1, 2):
        assert lib.jn_mx_linear_forward(p, p, p, None, many, 1, 1, kind, -1, p, p, all_, None) == 2
        assert b"too many outputs" in lib.jn_last_error()
        assert lib.jn_mx_linear_forward(p, p, p, None, many, 1, 1, kind, 1, p, p, all_, None) == 2
        assert lib.jn_mx_linear_backward(p, p, p, many, 1, 1, kind, p, p, all_, None) == 2
        assert lib.jn_mx_linear_backward(p, p, p, many, 8, 8, kind, p, p, all_, None) == 2
    assert lib.jn_mx_weight_grad(p, p, p, 1, (1 << 24) - 1, (1 << 24) - 1, 1, p, p, p, all_, None) == 2
