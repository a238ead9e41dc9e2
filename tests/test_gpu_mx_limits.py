"""Microscaled operators on more runs than one launch has threads for, and at the limits of the products."""

import pytest
import torch

import mx_exact as X
import step_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _memory(dev):
    yield
    torch.cuda.empty_cache()


def _need(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory")


# four threads a run: the second launch begins at row 2^29, the 2^32th thread is at row 2^30
ROWS = (1 << 30) + 1001
PLACES = (0, (1 << 29) - 2, 1 << 30, ROWS - 3)


def _narrow(dev):
    """[ROWS, 1] bf16, three rows of numbers at each place among zeros."""
    x = torch.zeros(ROWS, 1, dtype=torch.bfloat16, device=dev)
    for i, at in enumerate(PLACES):
        x[at:at + 3, 0] = torch.tensor([1.5 + i, -0.375, 7.0], dtype=torch.bfloat16)
    return x


@pytest.mark.parametrize("form", ["e4m3", "e2m1"])
def test_quantize_more_than_2_32_threads(dev, form):
    import jakal_net as J

    _need(48)
    x = _narrow(dev)
    q = J.mx_quantize(x, form)
    back = J.mx_dequantize(q)
    for at in PLACES:
        alone = J.mx_quantize(x[at:at + 3].clone(), form)
        assert torch.equal(q.codes[at:at + 3], alone.codes) and torch.equal(q.scales[at:at + 3], alone.scales)
        assert torch.equal(back[at:at + 3], J.mx_dequantize(alone))
    # the rows between are zeros everywhere: their least scale, and only the twelve others differ
    assert int((q.scales != 1).sum()) == 12 and int((back != 0).sum()) == 12


def test_gelu_more_than_2_32_threads(dev):
    import jakal_net as J

    _need(56)
    x = _narrow(dev).requires_grad_()
    y = J.gelu(x, saved="e4m3")
    grad, = torch.autograd.grad(y, x, torch.ones(1, dtype=torch.bfloat16, device=dev).expand(ROWS, 1))
    for at in PLACES:
        part = x.detach()[at:at + 3].clone().requires_grad_()
        alone = J.gelu(part, saved="e4m3")
        assert torch.equal(y.detach()[at:at + 3], alone.detach())
        assert torch.equal(grad[at:at + 3], torch.autograd.grad(alone.sum(), part)[0])
    assert int((y.detach() != 0).sum()) == 12 and int((grad != 0.5).sum()) == 12


def test_quantize_whole_runs_of_more_than_2_32_threads(dev):
    """64 GiB of bf16 in rows of whole runs."""
    import jakal_net as J

    _need(100)
    rows, dim = (1 << 20) + 3, 1 << 15
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device=dev)
    places = (0, (1 << 19) - 1, 1 << 20, rows - 2)
    for i, at in enumerate(places):
        x[at:at + 2].normal_(generator=torch.Generator(device=dev).manual_seed(i))
    q = J.mx_quantize(x, "e2m1")
    for at in places:
        alone = J.mx_quantize(x[at:at + 2].clone(), "e2m1")
        assert torch.equal(q.codes[at:at + 2], alone.codes) and torch.equal(q.scales[at:at + 2], alone.scales)
    # the other rows are zeros, whose scale is the least (the last two places share a row)
    written = sorted({at + i for at in places for i in (0, 1)})
    assert len(written) == 7 and int((q.scales != 1).sum()) == int((q.scales[written] != 1).sum()) == 7 * dim // 32


def test_products_beyond_a_grid_are_declined(dev):
    """2^24 tiles of 256 threads: a NotImplementedError, as for every call that the library has no kernel for."""
    import jakal_net as J

    _need(40)
    x, weight = torch.zeros((1 << 31) - 1, 1, device=dev), J.mx_quantize(torch.ones(1, 1, device=dev), "e2m1")
    with pytest.raises(NotImplementedError, match="too many outputs"):
        J.mx_linear(x, weight)
    with pytest.raises(NotImplementedError, match="too many outputs"):
        torch.ops.jakal_net_hip.mx_input_grad(x, weight.codes, weight.scales, 1)


@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_every_element_of_products_past_32_bits(dev, dtype):
    """2.29e9 outputs, and gradients of as many: whole numbers, each result against float64."""
    import jakal_net as J

    _need(60)
    kind, ops = O.DTYPES[dtype], torch.ops.jakal_net_hip
    rows, dim, out = 140_003, 64, 16_384
    chunks = [slice(at, min(rows, at + 10_000)) for at in range(0, rows, 10_000)]
    w, x = X.kept(1, out, dim, "e2m1", dev), X.kept(2, rows, dim, "e2m1", dev)
    weight = J.mx_quantize(w, "e2m1")
    for acts in (None, "e2m1"):
        y = J.mx_linear(x.to(kind), weight, activations=acts)
        for at in chunks:
            X.same(f"y of {acts}, rows from {at.start}", y[at], X.product(x[at], w.t()))
        del y
    g = torch.empty(rows, out, device=dev, dtype=kind)
    for i, at in enumerate(chunks):
        g[at] = X.whole(3 + i, at.stop - at.start, out, dev=dev, top=1).to(kind)
    gx = ops.mx_input_grad(g, weight.codes, weight.scales, dim)
    k = X.kept(4, rows, dim, "e4m3", dev)
    gw, gb = ops.mx_weight_grad(g, *ops.mx_codes(k, 0), dim, True)
    sums = ops.column_sums(g)
    want, size, bias = 0.0, 0.0, 0.0
    for at in chunks:
        part, kept = g[at].double(), k[at].double()
        X.same(f"grad_x, rows from {at.start}", gx[at], X.product(part, w))
        want, size, bias = want + part.t() @ kept, size + part.abs().t() @ kept.abs(), bias + part.sum(0)
        del part
    assert float(size.max()) < 2.0 ** 24  # sums that fp32 holds whatever their order
    X.same("grad_w", gw, want)
    X.same("grad_b", gb, bias)
    X.same("sums", sums, bias)
