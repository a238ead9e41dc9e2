"""That GELU's bounds see a tail that is not there, or not the function's."""

import math

import pytest
import torch

import gelu_tail as G
import step_oracle as O


def test_the_oracle_keeps_its_digits():
    """Against the asymptotic series of the tail, off by less than its next term."""
    for x in (-8.0, -10.0, -13.0, -20.0):
        z = x * x
        want = math.exp(-z / 2) / math.sqrt(2 * math.pi) / -x * (1 - 1 / z + 3 / z ** 2 - 15 / z ** 3 + 105 / z ** 4)
        assert abs(float(G.cdf(torch.tensor(x))) / want - 1) < 945 / z ** 5 + 1e-13


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_planted_mistakes_are_seen(kind):
    x = G.every(kind)
    value, bound = G.gelu(x)
    bound = bound + O.half(kind) * value.abs() + O.floor(kind)
    O.close("the function", value.to(kind), value, bound)
    for mistake in (torch.where(x < -5, 0.0, value), torch.where(x < -5, -value, value),
                    torch.where(x < -3, value * 1.02, value), torch.where(x > 5, value * 1.02, value)):
        with pytest.raises(AssertionError, match="times its bound"):
            O.close("a mistake", mistake.to(kind), value, bound)
    k = G.kept(kind)
    g = torch.ones_like(k)
    value, bound = G.slope(k, g)
    bound = bound + O.half(kind) * value.abs() + O.floor(kind)
    O.close("the slope", value.to(kind), value, bound)
    for mistake in (torch.where(k < -5, 0.0, value), torch.where(k < -3, value * 1.02, value)):
        with pytest.raises(AssertionError, match="times its bound"):
            O.close("a mistake", mistake.to(kind), value, bound)
