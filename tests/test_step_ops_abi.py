"""Sizes and limits that the training-step operators' C ABI states on the host."""

import ctypes

import pytest


def _lib():
    import jakal_net_native as jn

    return jn._LIB


@pytest.mark.parametrize("rows,dim", [(512, 262144), (100, 8193), (9, 33000), (1 << 20, 8200)])
def test_norm_workspace_of_wide_rows_is_its_slabs(rows, dim):
    """Rows beyond 8,192 elements are summed by slabs of 16 rows or more, 64 at most."""
    slabs = min(64, (rows + 15) // 16)
    assert _lib().jn_layer_norm_backward_workspace_bytes(rows, dim) == slabs * 2 * dim * 4


@pytest.mark.parametrize("dim", [1, 8, 100, 512, 1000, 4096, 8192])
def test_norm_workspace_of_register_rows_is_its_workgroups(dim):
    """One row of partial sums a workgroup, which has 256 threads at least and takes a row by 16 to 1024 of them."""
    threads = 16
    while dim > 8 * threads:
        threads *= 2
    for rows in (1, 4, 70, 1000, 2047, 2048, 70000, 1 << 24):
        parts, rest = divmod(_lib().jn_layer_norm_backward_workspace_bytes(rows, dim), 2 * dim * 4)
        assert rest == 0 and 1 <= parts <= min(512, -(-rows // max(1, 256 // threads)))


def test_loss_reduction_checks():
    lib = _lib()
    p = ctypes.c_void_p(4096)  # never read: every call below fails
    size = lib.jn_cross_entropy_reduce_workspace_bytes
    assert [size(n) for n in (-1, 0, 1, 32768)] == [0] * 4 and size(32769) == 9 * 16 and size(1 << 40) == 256 * 16

    def call(loss=p, target=p, rows=100000, reduction=2, reduced=p, count=p, ws=p, ws_bytes=1 << 20):
        return lib.jn_cross_entropy_reduce(loss, target, rows, -100, reduction, reduced, count, ws, ws_bytes, None)

    for bad in (dict(loss=None), dict(target=None), dict(rows=0), dict(rows=(1 << 40) + 1), dict(reduction=0),
                dict(reduction=3), dict(reduced=None), dict(count=None)):
        assert call(**bad) == 1, bad
    for bad in (dict(ws=None), dict(ws_bytes=size(100000) - 1)):
        assert call(**bad) == 4, bad


@pytest.mark.parametrize("dim,step", [(64, 32), (512, 8), (4096, 1), (8192, 1)])
def test_norm_rows_of_two_steps_stay_in_one_workgroup(dim, step):
    """step: the rows that a workgroup of 512 threads (1024 for the widest) has at a time."""
    size = _lib().jn_layer_norm_backward_workspace_bytes
    one = 2 * dim * 4
    assert size(1, dim) == size(2 * step, dim) == one and size(2 * step + 1, dim) > one
