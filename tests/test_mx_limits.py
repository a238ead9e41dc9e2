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


def _fake(*shape, dtype=torch.bfloat16, grad=False):
    return torch.empty(*shape, device="cuda", dtype=dtype, requires_grad=grad)


def test_sizes_beyond_the_library_are_declined_where_they_are_asked():
    """In the forward, though it is the backward's kernels that have no such size, and so that "kernel" takes the
    PyTorch form."""
    import jakal_net as J
    from torch._subclasses.fake_tensor import FakeTensorMode

    wide, many = 1 << 24, 1 << 31
    with FakeTensorMode():
        weight = J.MXTensor(_fake(5, 16, dtype=torch.uint8), _fake(5, 1, dtype=torch.uint8), "e2m1", 7)
        outs = J.MXTensor(_fake(wide, 16, dtype=torch.uint8), _fake(wide, 1, dtype=torch.uint8), "e2m1", 7)
        ins = J.MXTensor(_fake(5, wide // 2, dtype=torch.uint8), _fake(5, wide // 32, dtype=torch.uint8), "e2m1", wide)
        long = J.MXTensor(_fake(many // 2, dtype=torch.uint8), _fake(many // 32, dtype=torch.uint8), "e2m1", many)
        calls = [
            (lambda m: J.mx_dequantize(long, implementation=m), (many,)),
            (lambda m: J.mx_quantize(_fake(many), implementation=m).codes, (many,)),
            (lambda m: J.gelu(_fake(many, grad=True), saved="e4m3", implementation=m), (many,)),
            (lambda m: J.linear(_fake(2, 7), _fake(wide, 7, grad=True), saved="e4m3", implementation=m), (2, wide)),
            (lambda m: J.linear(_fake(2, wide), _fake(5, wide, grad=True), saved="e4m3", implementation=m), (2, 5)),
            (lambda m: J.linear(_fake(many, 7), _fake(5, 7, grad=True), saved="e4m3", implementation=m), (many, 5)),
            (lambda m: J.linear(_fake(many, 7), _fake(5, 7), _fake(5, grad=True), saved="e4m3", implementation=m), (many, 5)),
            (lambda m: J.mx_linear(_fake(many, 7), weight, implementation=m), (many, 5)),
            (lambda m: J.mx_linear(_fake(2, 7), outs, implementation=m), (2, wide)),
            (lambda m: J.mx_linear(_fake(2, wide), ins, activations="e2m1", implementation=m), (2, 5)),
        ]
        for i, (call, shape) in enumerate(calls):
            with pytest.raises(NotImplementedError):
                call("native")
            assert call("kernel").shape == shape, i
        # one less of each is taken, and a layer without a gradient of its weight is the plain one
        for call, shape in (
                (lambda: J.mx_quantize(_fake(many - 1)).scales, (many // 32,)),
                (lambda: J.gelu(_fake(many - 1, grad=True), saved="e4m3"), (many - 1,)),
                (lambda: J.linear(_fake(2, 7), _fake(wide - 1, 7, grad=True), saved="e4m3"), (2, wide - 1)),
                (lambda: J.linear(_fake(many - 1, 7), _fake(5, 7, grad=True), saved="e4m3"), (many - 1, 5)),
                (lambda: J.linear(_fake(many, 7, grad=True), _fake(5, 7), saved="e4m3"), (many, 5)),
                (lambda: J.mx_linear(_fake(many - 1, 7), weight), (many - 1, 5))):
            assert call().shape == shape
