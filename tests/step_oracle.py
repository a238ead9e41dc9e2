"""Float64 forms of the training-step operators, and how far fp32 may be from them.

Each function returns values and bounds: the bounds count roundings of half an
ulp (U = 2^-24 relative for fp32; ``half`` for the output type) on the terms
that the formulas sum, with ``depth`` roundings for a sum of n terms taken by 64
lanes or more and joined by a tree: n / 64 + 16.
"""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def floor(dtype) -> float:
    """Half the spacing of the type's smallest numbers (fp32 results may flush theirs to 0)."""
    if dtype is torch.float32 or dtype is torch.bfloat16:
        return 2.0 ** -126
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def depth(n: int) -> float:
    return n / 64 + 16


def close(what, got, want, bound) -> None:
    """|got - want| <= bound elementwise; NaN and infinities have to be where want has them."""
    got = got.detach().double().cpu()
    want, bound = want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} for {tuple(want.shape)}"
    if not got.numel():
        return
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)]), f"{what}: infinities"
    err = (got - want).abs()[finite]
    worst = float((err / bound[finite].clamp_min(1e-300)).max()) if err.numel() else 0.0
    print(f"{what}: largest error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, f"{what}: error {worst:.3f} times its bound"


def norm(x, weight, bias, eps, scale=1.0, g=None):
    """y of layer norm over scale * x and, with g, its gradients: {name: (value, bound)}.
    x [rows, dim] and g as the operator gets them; bounds before the output's own rounding."""
    v = x.double() * scale
    rows, dim = v.shape
    n = depth(dim)
    m = v.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((v - m) ** 2).mean(-1, keepdim=True) + eps)
    h = (v - m) * r
    top = v.abs().amax(-1, keepdim=True)
    # v and the mean are off by U and n U of the row's largest element; r by half of what the variance is
    # (n + 6 roundings of its own, and the centred values' error), against the value's own size
    e_c = (n + 3) * U * top
    e_r = (n + 8) * U + e_c * r
    e_h = e_c * r + h.abs() * e_r
    w = torch.ones(dim, dtype=torch.float64, device=v.device) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    out = {"y": (h * w + b, e_h * w.abs() + 2 * U * ((h * w).abs() + b.abs()))}
    if g is None:
        return out
    g = g.double()
    gw = g * w
    s1, s2 = gw.mean(-1, keepdim=True), (gw * h).mean(-1, keepdim=True)
    e_1 = n * U * gw.abs().mean(-1, keepdim=True)
    e_2 = n * U * (gw * h).abs().mean(-1, keepdim=True) + (gw.abs() * e_h).mean(-1, keepdim=True)
    inner = gw - s1 - h * s2
    e_in = 3 * U * (gw.abs() + s1.abs() + (h * s2).abs()) + e_1 + h.abs() * e_2 + e_h * s2.abs()
    out["grad_x"] = (scale * r * inner, abs(scale) * r * (e_in + inner.abs() * (e_r + 4 * U)))
    out["grad_weight"] = ((g * h).sum(0), (g.abs() * e_h).sum(0) + (depth(rows * 64) + 2) * U * (g * h).abs().sum(0))
    out["grad_bias"] = (g.sum(0), depth(rows * 64) * U * g.abs().sum(0))
    return out


def state(s, scale, g=None):
    v = s.double() * scale
    t = torch.tanh(v)
    # tanh's slope times its argument's rounding, and the function's own error (4 ulp)
    out = {"state": (t, U * (v.abs() * (1 - t * t) + 8 * t.abs()))}
    if g is not None:
        slope = 1.0 / torch.cosh(v.clamp(-300, 300)) ** 2
        d = scale * slope * g.double()
        # exp(-2 |v|) turns its argument's rounding into a relative error
        out["grad_state"] = (d, d.abs() * U * (4 * v.abs() + 24))
    return out


def cross_entropy(z, target, ignore=-100, reduction="mean", g=None):
    """Loss and gradient: {name: (value, bound)}; g: the incoming gradient (1 where none)."""
    z = z.double()
    rows, classes = z.shape
    valid = target != ignore
    inside = (target >= 0) & (target < classes)
    at = torch.where(inside, target, 0).unsqueeze(-1)
    top = z.amax(-1, keepdim=True)
    away = (z - top).abs()
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    log = torch.log(total)
    p = e / total
    # each exponential: 4 roundings of its argument (which is 0 where it counts most) and 4 of its own
    spread = torch.where(p > 0, p * away, 0.0).sum(-1, keepdim=True)
    e_log = U * (depth(classes) + 4 + 4 * spread + log.abs())
    zt = z.gather(-1, at)
    raw = (log + (top - zt)).squeeze(-1)
    e_raw = (e_log + 2 * U * ((top - zt).abs() + log)).squeeze(-1)
    nan = torch.full_like(raw, float("nan"))
    loss = torch.where(valid, torch.where(inside, raw, nan), 0.0)
    e_loss = torch.where(valid, e_raw, 0.0)
    count = valid.sum().double()
    if reduction == "none":
        out = {"loss": (loss, e_loss + U * loss.abs())}
    else:
        div = count if reduction == "mean" else 1.0
        out = {"loss": (loss.sum() / div, (e_loss.sum() + U * loss.abs().sum()) / div + 2 * U * (loss.sum() / div).abs())}
    scale = torch.ones((), dtype=torch.float64, device=z.device) if g is None else g.double()
    c = (scale / count if reduction == "mean" else scale).expand(rows).unsqueeze(-1)
    hot = torch.zeros_like(p).scatter_(-1, at, 1.0)
    d = (p - hot) * c
    e_p = torch.where(p > 0, p * (U * (4 * away + 8) + e_log + 2 * U * log.abs()), 0.0)
    bad = valid & ~inside
    d = torch.where(bad.unsqueeze(-1), float("nan"), d)
    d = torch.where(valid.unsqueeze(-1), d, 0.0)
    out["grad"] = (d, torch.where(valid.unsqueeze(-1), c.abs() * (e_p + 4 * U * (p - hot).abs()), 0.0))
    return out


def grads_norm(grads, kind=2.0) -> float:
    if kind == 2.0:
        return math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads))
    return max((float(t.double().abs().max()) for t in grads if t.numel()), default=0.0)
