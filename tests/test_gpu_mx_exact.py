"""Products with a microscaled operand on numbers whose sums are exact (tests/mx_exact.py):
equality with float64 over every kernel, tile and split, to sums of 131,072 terms."""

import ctypes

import pytest
import torch

import mx_exact as X
import step_oracle as O

pytestmark = pytest.mark.gpu

TYPES = list(O.DTYPES)
# Outputs [m, n] of sums over r: few rows, all tiles of bf16 with whole sums and split ones, rows that are
# no whole packs, ends inside runs, slices and tiles.
SIZES = [(1, 5, 33), (1, 16384, 2048), (7, 2056, 8192), (16, 300, 4099), (40, 1000, 16384), (64, 2048, 512), (65, 130, 96),
         (72, 72, 72), (72, 72, 520), (72, 520, 16392), (72, 1000, 8200), (72, 72, 128), (129, 257, 383), (136, 520, 8192),
         (152, 4104, 8200), (200, 16392, 72), (200, 16390, 256), (128, 2048, 16384), (300, 514, 288), (520, 4104, 4360),
         (1000, 8200, 72), (1024, 2048, 2048), (1531, 383, 4099), (1544, 2056, 72), (1536, 2056, 384), (2050, 700, 64),
         (8, 2048, 131072), (256, 256, 16384), (300, 520, 16392), (2000, 136, 4104)]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import jakal_net_native  # noqa: F401  (fails loudly when the library is missing)

    return torch.device("cuda:0")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,r", SIZES)
def test_forward(dev, m, n, r, dtype):
    import jakal_net as J

    kind = O.DTYPES[dtype]
    w = X.kept(1, n, r, "e2m1", dev)
    weight, bias = J.mx_quantize(w, "e2m1"), X.whole(2, n, dev=dev)
    assert torch.equal(J.mx_dequantize(weight), w)
    x, y = X.whole(3, m, r, dev=dev), X.kept(4, m, r, "e2m1", dev)
    X.same("plain x", J.mx_linear(x.to(kind), weight, bias.to(kind)), X.product(x, w.t(), bias))
    X.same("e2m1 x", J.mx_linear(y.to(kind), weight, bias.to(kind), activations="e2m1"), X.product(y, w.t(), bias))
    one = X.lonely(5, m, r, kind, 22, dev)  # two bits more of the weight's
    X.same("single elements", J.mx_linear(one, weight), X.product(one, w.t()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,r", SIZES)
def test_input_grad(dev, m, n, r, dtype):
    import jakal_net as J

    kind = O.DTYPES[dtype]
    w = X.kept(1, r, n, "e2m1", dev)
    weight = J.mx_quantize(w, "e2m1")
    for what, g in (("grad_x", X.whole(3, m, r, dev=dev)), ("single elements", X.lonely(5, m, r, kind, 22, dev))):
        got = torch.ops.jakal_net_hip.mx_input_grad(g.to(kind), weight.codes, weight.scales, n)
        X.same(what, got, X.product(g, w))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,r", SIZES)
def test_weight_grad(dev, m, n, r, dtype):
    kind = O.DTYPES[dtype]
    x = X.kept(1, r, n, "e4m3", dev)
    codes, scales = torch.ops.jakal_net_hip.mx_codes(x, 0)
    assert torch.equal(torch.ops.jakal_net_hip.mx_values(codes, scales, 0, n, torch.float32), x)
    # (single elements: the kept value has four bits)
    for what, g in (("grad_w", X.whole(3, r, m, dev=dev)), ("single elements", X.lonely(5, m, r, kind, 20, dev).t())):
        g = g.to(kind).contiguous()
        gw, gb = torch.ops.jakal_net_hip.mx_weight_grad(g, codes, scales, n, True)
        X.same(what, gw, X.product(g.t(), x))
        X.same(what + " of the bias", gb, g.double().sum(0))
        X.same(what + " of the bias alone", torch.ops.jakal_net_hip.column_sums(g), g.double().sum(0))


@pytest.mark.parametrize("m,n,r", [(16, 8, 8), (33, 1000, 256), (72, 72, 512), (72, 520, 16392), (200, 16392, 72),
                                   (1544, 2056, 72), (64, 1000, 8200), (1, 520, 16384), (2000, 4104, 136), (256, 256, 16384),
                                   (300, 520, 16392), (8, 2048, 131072), (1024, 2048, 16384)])
def test_linear_input_grad(dev, m, n, r):
    """The bf16 input gradient of a plain linear layer, where it has a kernel here."""
    import jakal_net_native as jn

    assert ctypes.CDLL(str(jn.library_path())).jn_linear_input_grad_fits(*map(ctypes.c_int64, (m, n, r)), 1) == 1
    w = X.whole(1, r, n, dev=dev)
    for what, g in (("grad_x", X.whole(3, m, r, dev=dev)), ("single elements", X.lonely(5, m, r, torch.bfloat16, 8, dev))):
        X.same(what, torch.ops.jakal_net_hip.linear_input_grad(g.bfloat16(), w.bfloat16()), X.product(g, w))


@pytest.mark.parametrize("acts", [None, "e2m1"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 17, 32, 33, 64])
def test_few_rows_give_an_output_the_same_bits_however_many_there_are(dev, rows, dtype, acts):
    """Tiles of outputs are shared out by how many there are; a sum's order is not."""
    import jakal_net as J

    kind = O.DTYPES[dtype]
    g = torch.Generator(device=dev).manual_seed(rows)
    w, x = torch.randn(17000, 2048, generator=g, device=dev), torch.randn(rows, 2048, generator=g, device=dev).to(kind)
    most = J.mx_linear(x, J.mx_quantize(w, "e2m1"), activations=acts)
    for outs in (16000, 10256, 10225, 8192, 4097, 300, 16):
        some = J.mx_linear(x, J.mx_quantize(w[:outs], "e2m1"), activations=acts)
        assert torch.equal(some, most[:, :outs]), outs
