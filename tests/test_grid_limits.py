"""Calls of more threads than a grid has along an axis (2^32) are declined before a launch, which would leave
outputs unwritten without an error."""

import ctypes

import pytest
import torch


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are no memory, should a call not be declined")
def test_more_threads_than_a_grid_has():
    import jakal_net_native as jn

    lib, p, f = jn._LIB, ctypes.c_void_p(4096), ctypes.c_float(1e-6)
    # a thread an element, a wave a row
    assert lib.jn_softsign_backward(p, p, (1 << 32) - 255, p, None) == 2
    assert lib.jn_softmax_backward(p, p, (1 << 26) - 3, 4, p, None) == 2
    assert lib.jn_unit_scale_forward(p, 1 << 26, 4, f, p, None) == 1
    assert lib.jn_unit_scale_backward(p, p, 1 << 26, 4, f, p, None) == 1
