"""The exponentials of the vocabulary loss's gradient, through the C ABI with
statistics that make the gradient a bare exponential."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("rows,classes", [(3, 700), (1100, 1500), (5, 4099), (4, 16384)])
def test_exponentials_to_two_units_in_the_last_place(rows, classes, shift):
    """With M = L = 0 and a gradient of 1 the classes beside the target get exp(z): two ulps of it, whatever z is
    (an exponential whose argument is rounded again is off by |z| / 2 of them)."""
    import jakal_net_native as jn

    gen = torch.Generator("cuda").manual_seed(classes)
    z = torch.rand(rows, classes, device="cuda", generator=gen) * -85.0
    target = torch.zeros(rows, device="cuda", dtype=torch.int64)
    stats, count, grad = (torch.full((n,), v, device="cuda") for n, v in ((2 * rows, 0.0), (1, 1.0), (1, 1.0)))
    # shift: the gradient's rows do not start on 16 bytes where the logits' do
    out = torch.empty(rows * classes + shift, device="cuda")[shift:].view(rows, classes)
    rc = jn._LIB.jn_cross_entropy_backward(*(ctypes.c_void_p(t.data_ptr()) for t in (z, target, stats, count, grad)),
                                           rows, classes, -100, 1, 0, ctypes.c_void_p(out.data_ptr()),
                                           ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    want = torch.exp(z.double())[:, 1:]
    worst = float(((out[:, 1:].double() - want).abs() / want).max()) / 2.0 ** -23
    print(f"{rows} x {classes}: {worst:.2f} ulps", flush=True)
    assert worst <= 2.0
