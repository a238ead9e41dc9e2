"""Float64 forms of the operators on microscaled numbers, and how far fp32 may be
from them (bounds as in step_oracle: U = 2^-24, before the output's own rounding)."""

from __future__ import annotations

import math

import torch

from step_oracle import U, depth

RUN = 32


def magnitudes(form: str) -> torch.Tensor:
    """The format's magnitudes by code."""
    if form == "e2m1":
        return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    out = []
    for code in range(127):
        e, m = code >> 3, code & 7
        out.append((1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6)
    return torch.tensor(out, dtype=torch.float64)


def quantize(x: torch.Tensor, form: str):
    """(values in float64, element codes, scale codes) of x [..., size]: a search for the
    nearest magnitude, ties to the even code, and for the smallest fitting power of two."""
    grid = magnitudes(form)
    x = x.detach().double().cpu()
    size = x.shape[-1]
    v = torch.nn.functional.pad(x, (0, -size % RUN)).unflatten(-1, (-1, RUN))
    most = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(most)
    most = torch.where(bad, 0.0, most)
    e = torch.full_like(most, -126.0)
    for _ in range(260):
        e = torch.where(most > grid[-1] * torch.exp2(e), e + 1, e)
    s = torch.where(bad, 0.0, v).abs() * torch.exp2(-e)
    middle = (grid[1:] + grid[:-1]) / 2
    # codes whose upper neighbour's border lies below: at a border, the even code of the two
    code = torch.searchsorted(middle, s.contiguous())
    at_border = (code < len(middle)) & (s == middle[code.clamp(max=len(middle) - 1)]) & (code % 2 == 1)
    code = torch.where(at_border, code + 1, code)
    sign = torch.signbit(v) & ~bad
    value = torch.where(sign, -grid[code], grid[code]) * torch.exp2(e)
    value = torch.where(bad, math.nan, value)
    top = 128 if form == "e4m3" else 8
    code = torch.where(bad, 0x7F if form == "e4m3" else 0, code + top * sign)
    scale = torch.where(bad, 255, (e + 127).long())
    return value.flatten(-2)[..., :size], code.flatten(-2), scale.squeeze(-1)


def packed(code: torch.Tensor, form: str) -> torch.Tensor:
    """Element codes as they lie in memory."""
    code = code.to(torch.uint8)
    return code if form == "e4m3" else code[..., 0::2] | (code[..., 1::2] << 4)


def product(a: torch.Tensor, b: torch.Tensor, bias=None):
    """a [m, k] @ b [k, n] + bias with exact products: (value, bound).  The sums are of k
    terms in an unknown order, each addition off by at most a whole unit (2^-23) of a
    partial sum, which the terms' magnitudes bound; the bias' addition by half a unit."""
    a, b = a.double(), b.double()
    value, size = a @ b, a.abs() @ b.abs()
    bound = 2 * U * a.shape[1] * size
    if bias is not None:
        value = value + bias.double()
        bound = bound + 2 * U * (size + bias.double().abs())
    return value, bound


def sums(g: torch.Tensor):
    """Sums over rows, in fp32 by whatever order."""
    g = g.double()
    return g.sum(0), U * g.shape[0] * g.abs().sum(0)


def gelu(x: torch.Tensor):
    """The error function and the exponential are off by 4 units of 1 at most, their
    argument by a rounding, which the function's slope (below 1.13) passes on."""
    x = x.double()
    size = x.abs()
    return x * torch.special.ndtr(x), size * U * (16 + 2 * size.clamp(max=9.0))


def gelu_slope(k: torch.Tensor, g: torch.Tensor):
    k, g = k.double(), g.double()
    dense = torch.exp(-k * k / 2) / math.sqrt(2 * math.pi)
    value = g * (torch.special.ndtr(k) + k * dense)
    # exp turns its argument's roundings into relative ones
    e = 16 + 2 * k.abs().clamp(max=9.0) + (k.abs() * dense) * (8 + 2 * k * k)
    return value, g.abs() * U * e


def centred(x: torch.Tensor) -> torch.Tensor:
    """x less its rows' means, fp32 numbers both."""
    return x.float() - x.double().mean(-1, keepdim=True).float()


def kept_norm(x, weight, eps, scale, g):
    """Gradients of layer norm over scale * x with h from the centred x in e4m3: {name: (value, bound)}."""
    v, k = x.double() * scale, quantize(centred(x), "e4m3")[0] * scale
    rows, dim = v.shape
    n = depth(dim)
    m = v.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((v - m) ** 2).mean(-1, keepdim=True) + eps)
    h = k * r
    # the statistics' errors are the plain norm's; what was kept is exact
    e_r = (n + 8) * U + (n + 3) * U * v.abs().amax(-1, keepdim=True) * r
    e_h = h.abs() * (e_r + 2 * U)
    w = torch.ones(dim, dtype=torch.float64, device=v.device) if weight is None else weight.double()
    g = g.double()
    gw = g * w
    s1, s2 = gw.mean(-1, keepdim=True), (gw * h).mean(-1, keepdim=True)
    e_1 = n * U * gw.abs().mean(-1, keepdim=True)
    e_2 = n * U * (gw * h).abs().mean(-1, keepdim=True) + (gw.abs() * e_h).mean(-1, keepdim=True)
    inner = gw - s1 - h * s2
    e_in = 3 * U * (gw.abs() + s1.abs() + (h * s2).abs()) + e_1 + h.abs() * e_2 + e_h * s2.abs()
    return {"grad_x": (scale * r * inner, abs(scale) * r * (e_in + inner.abs() * (e_r + 4 * U))),
            "grad_weight": ((g * h).sum(0),
                            (g.abs() * e_h).sum(0) + (depth(rows * 64) + 2) * U * (g * h).abs().sum(0)),
            "grad_bias": (g.sum(0), depth(rows * 64) * U * g.abs().sum(0))}
