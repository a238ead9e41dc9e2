"""The layer norm's parameter gradients over many rows, exactly: rows of +1 and -1
with eps = 0 have h = +1 and -1, and gradients of small whole numbers then have
column sums below 2^24, which fp32 holds in any order.  A row that is lost, read
twice or read from elsewhere shows as a whole number."""

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


@pytest.mark.parametrize("rows,dim,dtype,offset", [
    (1, 64, "fp32", 0), (129, 64, "fp32", 0), (2047, 100, "fp16", 0), (2050, 384, "bf16", 1), (9001, 1000, "fp32", 0),
    (9001, 1002, "bf16", 0), (4099, 1536, "bf16", 0), (70000, 24, "fp32", 0), (1031, 8192, "fp32", 0),
    (1031, 8200, "fp32", 0), (33, 8200, "bf16", 1), (5000, 9002, "fp16", 0), ((1 << 21) + 3, 1024, "bf16", 0),
    ((1 << 25) + 5, 64, "bf16", 0), ((1 << 21) + 3, 1026, "bf16", 0), (300001, 8200, "bf16", 0)])
def test_column_sums_are_exact(dev, rows, dim, dtype, offset):
    import jakal_net as J

    kind = O.DTYPES[dtype]
    gen = torch.Generator(dev).manual_seed(rows + dim)

    def made():
        return torch.empty(offset + rows * dim, device=dev, dtype=kind)[offset:].view(rows, dim)

    x, g = made(), made()
    signs = torch.randint(0, 2, (rows, 1), device=dev, generator=gen).mul(2).sub(1).to(kind)
    pattern = torch.ones(dim, device=dev, dtype=kind)
    pattern[torch.randperm(dim, device=dev, generator=gen)[: dim // 2]] = -1
    torch.mul(signs, pattern, out=x)
    # column sums stay below 2^24: 0 to 7, or where that many rows could pass it, a 1 in every fourth place
    few = 7 * rows >= 1 << 24
    whole = torch.zeros(2, dim, device=dev, dtype=torch.float64)
    for x0, g0 in zip(x.split(1 << 16), g.split(1 << 16)):
        drawn = torch.randint(0, 4 if few else 8, g0.shape, device=dev, generator=gen, dtype=torch.int32)
        g0.copy_(drawn == 0 if few else drawn)
        g0[-1] = 1  # the chunk's last row, and so the last of all, counts in every column
        d = g0.double()
        whole[0] += (d * x0).sum(0)
        whole[1] += d.sum(0)
    assert 0 < float(whole[1].min()) and float(whole[1].max()) < 1 << 24
    w, b = (torch.ones(dim, device=dev).requires_grad_() for _ in range(2))
    y = J.layer_norm(x, w, b, eps=0.0)
    gw, gb = torch.autograd.grad(y, [w, b], g)
    assert torch.equal(gw.double(), whole[0]) and torch.equal(gb.double(), whole[1])
    # with the input gradient beside them they are the same sums
    leaf = x.requires_grad_()
    gx, gw, gb = torch.autograd.grad(J.layer_norm(leaf, w, b, eps=0.0), [leaf, w, b], g)
    assert torch.equal(gw.double(), whole[0]) and torch.equal(gb.double(), whole[1])
