"""GELU that keeps e4m3 in half precision, at every number of its types: in relative terms
below 0, where the function falls to 10^-43."""

import pytest
import torch

import gelu_tail as G
import step_oracle as O

pytestmark = pytest.mark.gpu
HALVES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


@pytest.mark.parametrize("dtype", list(HALVES))
def test_every_number(dev, dtype):
    import jakal_net as J

    kind = HALVES[dtype]
    x = G.every(kind)
    for keep in (False, True):
        y = J.gelu(x.to(dev).requires_grad_(keep), saved="e4m3")
        value, bound = G.gelu(x)
        O.close(dtype, y, value, bound + O.half(kind) * value.abs() + O.floor(kind))


@pytest.mark.parametrize("dtype", list(HALVES))
def test_slope_at_every_kept_number(dev, dtype):
    import jakal_net as J

    kind = HALVES[dtype]
    x = G.kept(kind).to(dev).requires_grad_()
    back = J.mx_dequantize(J.mx_quantize(x.detach()), torch.float32)
    assert torch.equal(back, x.detach().float())
    g = torch.linspace(0.5, 2.0, 32).to(kind).expand(x.shape)
    got, = torch.autograd.grad(J.gelu(x, saved="e4m3"), x, g.to(dev))
    value, bound = G.slope(x.detach().cpu(), g)
    O.close(dtype, got, value, bound + O.half(kind) * value.abs() + O.floor(kind))
