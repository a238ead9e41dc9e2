"""GELU and its slope in float64, with bounds in relative terms on the negative side, for
half precision's tail of the normal distribution:

    Phi(-|x|) = exp(-x^2 / 2) t Q(t) / 2,  t = 1 / (1 + |x| / sqrt 8)

U = 2^-24.  x^2 is exact (22 bits at most); its product with a constant is off by 2 U of
itself, which the exponential turns into x^2 U, and is off by 2 U itself.  t is off by 5 U
(two roundings and a constant in its denominator, the reciprocal's 2 U), which t Q(t)
passes on 2.3-fold.  Q's eight steps are off by 9 U of the sum of its terms' magnitudes,
which is 2.15 times itself at most (at t = 1), and Q by 7.4e-8 < 2 U.  With three products
behind it the tail is off by (x^2 + 2 + 12 + 20 + 2 + 3) U < (x^2 + 40) U of itself.
Above 0 the function is one less the tail."""

from __future__ import annotations

import math

import torch

from step_oracle import U


def cdf(x: torch.Tensor) -> torch.Tensor:
    """Phi in float64, in relative terms on both sides."""
    return 0.5 * torch.special.erfc(-x.double() / math.sqrt(2.0))


def gelu(x: torch.Tensor):
    x = x.double()
    tail = cdf(-x.abs())
    return x * cdf(x), x.abs() * U * ((x * x + 40) * tail + 3 * cdf(x))


def slope(k: torch.Tensor, g: torch.Tensor):
    """g (Phi + k phi): phi's own error is the exponential's and three roundings."""
    k, g = k.double(), g.double()
    part = k * torch.exp(-k * k / 2) / math.sqrt(2 * math.pi)
    bound = U * ((k * k + 40) * cdf(-k.abs()) + 3 * cdf(k) + (k * k + 8) * part.abs())
    return g * (cdf(k) + part), g.abs() * (bound + 2 * U * (cdf(k) + part).abs())


def every(dtype: torch.dtype) -> torch.Tensor:
    """Every finite number of a 16-bit type."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    return x[torch.isfinite(x)]


def kept(dtype: torch.dtype) -> torch.Tensor:
    """Rows of 32 of one number that e4m3 keeps as it is, of every significand, from 2^-12 to 15."""
    v = torch.tensor([(1 + m / 8) * 2.0 ** e for e in range(-12, 4) for m in range(8) if (1 + m / 8) * 2.0 ** e <= 15])
    return torch.cat([v, -v])[:, None].expand(-1, 32).to(dtype)
