"""The layer norm's backward through the C ABI with exactly the workspace that it
asks for, between guard bytes."""

import ctypes

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("rows,dim", [(4, 8), (70, 64), (300, 512), (2047, 100), (2050, 384), (70000, 24), (60, 8192),
                                      (33, 8200), (1030, 9001)])
def test_exact_workspace_between_guards(rows, dim, offset):
    import jakal_net_native as jn

    lib = jn._LIB
    gen = torch.Generator("cuda").manual_seed(rows + dim)

    def made():
        return torch.randn(offset + rows * dim, device="cuda", generator=gen)[offset:].view(rows, dim)

    x, g = made(), made()
    y, gx = torch.empty(rows, dim, device="cuda"), torch.empty(rows, dim, device="cuda")
    stats, gw, gb = (torch.empty(n, device="cuda") for n in (2 * rows, dim, dim))
    need = lib.jn_layer_norm_backward_workspace_bytes(rows, dim)
    guard = 4096
    ws = torch.full((guard + need + guard,), 171, device="cuda", dtype=torch.uint8)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def p(t, at=0):
        return ctypes.c_void_p(t.data_ptr() + at)

    assert lib.jn_layer_norm_forward(None, p(x), None, None, rows, dim, 1.0, 1e-5, 0, 0, 0, None, p(y), p(stats),
                                     stream) == 0
    assert lib.jn_layer_norm_backward(None, p(x), None, p(stats), None, p(g), rows, dim, 1.0, 0, 0, 0, None, p(gx), p(gw),
                                      p(gb), p(ws, guard), need, stream) == 0
    assert bool((ws[:guard] == 171).all()) and bool((ws[guard + need:] == 171).all())
    want = O.norm(x, None, None, 1e-5, 1.0, g)
    for name, got in (("y", y), ("grad_x", gx), ("grad_weight", gw), ("grad_bias", gb)):
        O.close(name, got, want[name][0], want[name][1] + O.U * want[name][0].abs())
