"""Layer norm of very wide rows on the HIP library: the launches that a backward
with parameter gradients needs up to 2^28 - 1 elements a row, and sums over the
row that keep their digits."""

import pytest
import torch

import step_oracle as O

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


def _sum_roundings(dim):
    """Roundings of a row's sum by 256 threads: a term's own few, runs of up to 256 terms in fp32 (their sums are
    joined in 64 bits) and a join of 256 threads."""
    return min(dim // 256, 256) + 12


@pytest.mark.parametrize("dim", [9000, (1 << 24) + 8, (1 << 26) + 3])
def test_constant_rows_stay_at_their_mean(dev, dim):
    """A row of one value: y is what the mean's roundings leave over sqrt(eps)."""
    import jakal_net as J

    x = torch.full((2, dim), 0.1, device=dev)
    x[1] = 0.7
    y = J.layer_norm(x, eps=1e-5)
    off = _sum_roundings(dim) * O.U * x.amax(-1, keepdim=True).double() / 1e-5 ** 0.5
    assert bool((y.double().abs() <= off).all()), float((y.double().abs() / off).max())


@pytest.mark.parametrize("dim", [9001, (1 << 24) + 8, (1 << 26) + 3])
def test_wide_rows_against_float64(dev, dim):
    """Positive terms in every sum (values and gradients above zero), where roundings of a long fp32 sum add up."""
    import jakal_net as J

    gen = torch.Generator(dev).manual_seed(dim)
    x = torch.rand(1, dim, device=dev, generator=gen).requires_grad_()
    g = torch.rand(1, dim, device=dev, generator=gen) + 0.5
    y = J.layer_norm(x)
    (gx,) = torch.autograd.grad(y, x, g)
    n, U = _sum_roundings(dim), O.U
    v, gd = x.detach().double(), g.double()
    m = v.mean()
    r = 1.0 / torch.sqrt(((v - m) ** 2).mean() + 1e-5)
    h = (v - m) * r
    # the mean is off by n U of its terms' mean, a centred value by a rounding more; the deviation by half of the
    # squares' n + 4 roundings and by the mean's error squared, which is nothing here
    e_c = n * U * float(v.mean()) + U
    e_r = (n / 2 + 4) * U
    e_h = e_c * r + h.abs() * (e_r + 2 * U)
    assert bool(((y.double() - h).abs() <= e_h + U * h.abs()).all())
    s1, s2 = gd.mean(), (gd * h).mean()
    e_1 = (n + 1) * U * s1
    e_2 = (n + 2) * U * (gd * h).abs().mean() + (gd * e_h).mean()
    inner = gd - s1 - h * s2
    e_in = 3 * U * (gd + s1 + (h * s2).abs()) + e_1 + h.abs() * e_2 + e_h * s2.abs()
    bound = r * (e_in + inner.abs() * (e_r + 4 * U))
    assert bool(((gx.double() - r * inner).abs() <= bound + U * (r * inner).abs()).all())
