"""Layer norm of very wide rows on the HIP library: the launches that a backward
with parameter gradients needs up to 2^28 - 1 elements a row."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


def _parameter_gradients(dev, rows, dim, dtype):
    """Gradients of rows of +1 and -1 in equal shares: mean 0, variance 1, all sums of it exact."""
    import jakal_net as J

    x = torch.ones(rows, dim, device=dev, dtype=dtype)
    x[:, 1::2] = -1
    if dim % 2:
        x[:, -1] = 0
    g = torch.randint(-8, 9, (rows, dim), device=dev, generator=torch.Generator(dev).manual_seed(dim)).to(dtype)
    w, b = (torch.ones(dim, device=dev).requires_grad_() for _ in range(2))
    gw, gb = torch.autograd.grad(J.layer_norm(x, w, b), [w, b], g)
    return x, g, gw, gb


@pytest.mark.parametrize("rows,dim,dtype", [(1, (1 << 25) - 16, torch.float32), (3, 1 << 25, torch.float32),
                                            (2, (1 << 25) + 8, torch.bfloat16), (2, (1 << 26) + 1, torch.float32),
                                            (1, (1 << 28) - 1, torch.bfloat16)])
def test_parameter_gradients_of_the_widest_rows(dev, rows, dim, dtype):
    x, g, gw, gb = _parameter_gradients(dev, rows, dim, dtype)
    # small whole numbers: the sums over the rows are exact
    assert torch.equal(gb, g.float().sum(0))
    # the variance is 1 or (dim - 1) / dim: h is x to within 1 / sqrt(1 + eps) and the 2^-24 of a few roundings
    want = (g.double() * x.double()).sum(0) / (1.0 + 1e-5) ** 0.5
    assert bool(((gw.double() - want).abs() <= (1 / dim + 8 * 2.0 ** -24) * (g.double() * x).abs().sum(0)).all())
