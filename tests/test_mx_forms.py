"""The PyTorch forms of the operators on microscaled numbers: values of one axis."""

import pytest
import torch

import mx_oracle as M
import step_oracle as O

MODES = ["reference", "streaming", "kernel", "native"]


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("acts", [None, "e2m1"])
def test_values_of_one_axis(mode, acts):
    """A bias' gradient of a single row is the output's gradient."""
    import jakal_net as J

    x, b, g = _rand(1, 50).requires_grad_(), _rand(3, 9).requires_grad_(), _rand(2, 9)
    weight, w = J.mx_quantize(_rand(4, 9, 50), "e2m1"), M.quantize(_rand(4, 9, 50), "e2m1")[0]
    y = J.mx_linear(x, weight, b, activations=acts, implementation=mode)
    assert y.shape == (9,)
    gx, gb = torch.autograd.grad(y, (x, b), g)
    assert torch.equal(gb, g)
    value, bound = M.product(g[None], w)
    O.close("grad_x", gx[None], value, bound + O.U * value.abs())
