"""That the products' exact tests see what a product loses: mistakes planted in float64."""

import pytest
import torch

import mx_exact as X
import step_oracle as O
from test_gpu_mx_exact import SIZES


@pytest.mark.parametrize("m,n,r", SIZES)
@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_lost_terms_are_seen(m, n, r, dtype):
    """The last eight terms, a slice of 64 in the middle, a half: each changes outputs in every type."""
    kind = O.DTYPES[dtype]
    m, n = min(m, 8), min(n, 33)
    operands = [(X.whole(3, m, r), X.kept(1, n, r, "e2m1").t()), (X.kept(4, m, r, "e2m1"), X.kept(1, n, r, "e2m1").t()),
                (X.whole(3, m, r), X.kept(1, r, n, "e2m1")), (X.whole(3, r, m).t(), X.kept(1, r, n, "e4m3"))]
    for a, b in operands:
        want = X.product(a, b)
        X.same("nothing lost", want.to(kind), want)
        for lost in (slice(max(0, r - 8), r), slice(r // 2 // 64 * 64, r // 2 // 64 * 64 + 64), slice(r // 2, r)):
            part = a.clone()
            part[:, lost] = 0
            with pytest.raises(AssertionError, match="differ"):
                X.same("lost", X.product(part, b).to(kind), want)


@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_lost_bits_are_seen(dtype):
    """fp32's and fp16's lower terms: a single element without the bits below bf16's."""
    kind = O.DTYPES[dtype]
    x, w = X.lonely(5, 64, 400, kind, 22), X.kept(1, 50, 400, "e2m1").t()
    want = X.product(x, w)
    assert torch.equal(want.float().double(), want)  # fp32 holds every product
    short = x.bfloat16().to(kind)
    if kind is torch.bfloat16:
        assert torch.equal(short, x)
    else:
        with pytest.raises(AssertionError, match="differ"):
            X.same("lost", X.product(short, w).to(kind), want)
    at = (x != 0).nonzero()[:, 1]
    assert {0, 399, 398, 392, 391, 32, 31, 64, 63, 128, 127, 256, 255} <= set(at.tolist())


@pytest.mark.parametrize("dtype", list(O.DTYPES))
def test_lost_rows_of_a_long_sum_are_seen(dtype):
    """A gradient over 140,003 rows: half of them gone, those past 2^31 elements of 16,384 columns, rows read twice."""
    kind, rows = O.DTYPES[dtype], 140_003
    g, k = X.whole(3, rows, 4, top=1), X.kept(4, rows, 64, "e4m3")
    want, sums = X.product(g.t(), k), g.double().sum(0)
    past = 2 ** 31 // 16_384
    for lost in (slice(0, rows // 2), slice(past, rows), slice(rows - 64, rows)):
        part = g.clone()
        part[lost] = 0
        with pytest.raises(AssertionError, match="differ"):
            X.same("lost", X.product(part.t(), k).to(kind), want)
        with pytest.raises(AssertionError, match="differ"):
            X.same("lost", part.double().sum(0).to(kind), sums)
    part = g.clone()
    part[past:] = g[:rows - past]
    with pytest.raises(AssertionError, match="differ"):
        X.same("wrapped", X.product(part.t(), k).to(kind), want)
