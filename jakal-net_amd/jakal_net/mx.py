"""Microscaled tensors: activations kept in 8 bits, products by 4-bit weights.

A microscaled tensor holds its last axis in runs of 32 elements (the last run may
be short), each run one power of two times short floats:

* ``"e4m3"``: 8 bits, largest 448; ``"e2m1"``: 4 bits, the magnitudes 0, 0.5, 1,
  1.5, 2, 3, 4 and 6;
* a run's scale is the smallest power of two, 2**-126 at least, that keeps its
  largest magnitude within the format; elements are rounded to the nearest value,
  ties to the even code.  A run with an infinity or a NaN is NaN as a whole.

``saved="e4m3"`` (``linear``, ``gelu``, and ``layer_norm`` and ``stabilize`` of
``jakal_net.norm``) keeps what the backward needs of the layer's input in e4m3,
1.03 bytes an element (the norms, what is left of it beside its mean).  The output
is that of the plain layer; the gradients are its formulas at the kept input.  ``mx_linear`` multiplies by a frozen e2m1 weight,
its activations as they are or microscaled in e2m1 on the way in.

``implementation`` as in the operators: ``"native"`` (the default here) runs the
HIP library for GPU tensors of fp32, bf16 or fp16 and raises where it cannot, CPU
tensors (and a native module without these operators) take the PyTorch form;
``"kernel"`` takes the PyTorch form where the library declines; ``"reference"`` and
``"streaming"`` are the PyTorch form.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import Tensor, nn
from torch.nn import functional as F

from jakal_net.core import ImplementationMode, check_implementation
from jakal_net.native_backend import native_op

RUN = 32
FORMATS = ("e4m3", "e2m1")
# largest exponent, largest significand, mantissa bits, smallest normal exponent
_SHAPES = {"e4m3": (8, 1.75, 3, -6), "e2m1": (2, 1.5, 1, 0)}


def check_format(format: str) -> None:
    if format not in FORMATS:
        raise ValueError(f"a microscaled format is one of {FORMATS}, got {format!r}.")


def check_activations(activations: str | None) -> None:
    if activations not in (None, "e2m1"):
        raise ValueError(f"activations are None (as they are) or 'e2m1', got {activations!r}.")


def check_saved(saved: str | None) -> None:
    if saved not in (None, "e4m3"):
        raise ValueError(f"saved is None (as it is) or 'e4m3', got {saved!r}.")


def _runs(size: int) -> int:
    return -(-size // RUN)


@dataclass(frozen=True)
class MXTensor:
    """A microscaled tensor of rows of ``size`` elements: ``codes [..., bytes]`` (32
    bytes a run of e4m3; 16 of e2m1, the first of two elements in the low half),
    ``scales [..., runs]`` (2**(s - 127); 255: NaN), both uint8.  ``dtype`` is the
    type it dequantises to by default."""

    codes: Tensor
    scales: Tensor
    format: str
    size: int
    dtype: torch.dtype = torch.float32

    def __post_init__(self) -> None:
        check_format(self.format)
        width = _runs(self.size) * (RUN if self.format == "e4m3" else RUN // 2)
        if (self.size < 1 or self.codes.dtype != torch.uint8 or self.scales.dtype != torch.uint8
                or self.codes.shape[-1:] != (width,) or self.scales.shape != (*self.codes.shape[:-1], _runs(self.size))):
            raise ValueError(f"{self.format} rows of {self.size} elements need uint8 codes [..., {width}] and scales "
                             f"[..., {_runs(self.size)}], got {tuple(self.codes.shape)} and "
                             f"{tuple(self.scales.shape)}.")

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.size))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def to(self, device) -> MXTensor:
        return MXTensor(self.codes.to(device), self.scales.to(device), self.format, self.size, self.dtype)


# ---------------------------------------------------------------------------
# PyTorch forms
# ---------------------------------------------------------------------------
def _two_to(exponents: Tensor) -> Tensor:
    """2**e in fp32 for -126 <= e <= 127."""
    return ((exponents.to(torch.int32) + 127) << 23).view(torch.float32)


def _check_real(what: str, x: Tensor) -> None:
    if x.is_complex():
        raise NotImplementedError(f"{what} takes real values, got {x.dtype}.")


def _quantize(x: Tensor, format: str) -> tuple[Tensor, Tensor]:
    _check_real("mx_quantize", x)
    top, significand, bits, least = _SHAPES[format]
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"mx_quantize needs a last axis of at least one element, got shape {tuple(x.shape)}.")
    v = F.pad(x.detach().float(), (0, -x.shape[-1] % RUN)).unflatten(-1, (-1, RUN))
    most = v.abs().amax(-1)
    finite = torch.isfinite(most)
    part, e = torch.frexp(torch.where(finite, most, 0.0))  # part in [0.5, 1)
    e = torch.where(part == 0, -126, e - 1 - top + (2.0 * part > significand)).clamp(min=-126)
    v = torch.where(finite.unsqueeze(-1), v, 0.0) * _two_to(-e).unsqueeze(-1)
    size = v.abs()
    exponent = ((size.view(torch.int32) >> 23) - 127).clamp(min=least)
    steps = torch.round(size / _two_to(exponent - bits)).to(torch.int32)  # of the binade's step; ties to even
    code = steps + ((exponent - least) << bits)
    sign = torch.signbit(v).to(torch.int32)
    code = (code | (sign << (7 if format == "e4m3" else 3))).to(torch.uint8)
    code = torch.where(finite.unsqueeze(-1), code, 0x7F if format == "e4m3" else 0).flatten(-2)
    if format == "e2m1":
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code, torch.where(finite, e + 127, 255).to(torch.uint8)


def _dequantize(codes: Tensor, scales: Tensor, format: str, size: int, dtype: torch.dtype) -> Tensor:
    _, _, bits, least = _SHAPES[format]
    if format == "e2m1":
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    code = codes.to(torch.int32)
    sign_at = 7 if format == "e4m3" else 3
    place = code & ((1 << sign_at) - 1)
    exponent = (place >> bits).clamp(min=1)
    significand = (place & ((1 << bits) - 1)) + torch.where(place >> bits > 0, 1 << bits, 0)
    value = significand.to(torch.float32) * _two_to(exponent - 1 + least - bits)
    if format == "e4m3":
        value = torch.where(place == 0x7F, math.nan, value)
    value = torch.where(code >> sign_at > 0, -value, value)
    s = scales.to(torch.int32)
    scale = torch.where(s == 255, math.nan, torch.where(s == 0, 2.0 ** -127, _two_to(s.clamp(1, 254) - 127)))
    return (value.unflatten(-1, (-1, RUN)) * scale.unsqueeze(-1)).flatten(-2)[..., :size].to(dtype)


def _wide(t: Tensor) -> Tensor:
    return t.float() if t.dtype in (torch.float16, torch.bfloat16) else t


class _MXLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scales, bias, activations):
        _check_real("mx_linear", x)
        ctx.save_for_backward(codes, scales)
        ctx.size, ctx.dtype = x.shape[-1], x.dtype
        v = x.float()
        if activations is not None:
            v = _dequantize(*_quantize(x, activations), activations, x.shape[-1], torch.float32)
        y = v @ _dequantize(codes, scales, "e2m1", x.shape[-1], torch.float32).t()
        return (y if bias is None else y + bias.float()).to(x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        g = grad.float()
        gx = gb = None
        if ctx.needs_input_grad[0]:
            gx = (g @ _dequantize(*ctx.saved_tensors, "e2m1", ctx.size, torch.float32)).to(ctx.dtype)
        if ctx.needs_input_grad[3]:
            gb = g.reshape(-1, g.shape[-1]).sum(0).to(ctx.dtype)
        return gx, None, None, gb, None


class _LinearSaved(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(*_quantize(x, "e4m3"), weight)
        return F.linear(x, weight, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        codes, scales, weight = ctx.saved_tensors
        g = _wide(grad)
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            gx = (g @ _wide(weight)).to(weight.dtype)
        rows = g.reshape(-1, g.shape[-1])
        if ctx.needs_input_grad[1]:
            kept = _dequantize(codes, scales, "e4m3", weight.shape[1], rows.dtype).reshape(-1, weight.shape[1])
            gw = (rows.t() @ kept).to(weight.dtype)
        if ctx.needs_input_grad[2]:
            gb = rows.sum(0).to(weight.dtype)
        return gx, gw, gb


class _GELUSaved(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(*_quantize(x, "e4m3"))
        ctx.size = x.shape[-1]
        return F.gelu(x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        k = _dequantize(*ctx.saved_tensors, "e4m3", ctx.size, torch.float32)
        slope = 0.5 * (1.0 + torch.erf(k * math.sqrt(0.5))) + k * torch.exp(-0.5 * k * k) / math.sqrt(2.0 * math.pi)
        return (_wide(grad) * slope).to(grad.dtype)


class _NormSaved(torch.autograd.Function):
    """The layer norm of scale * x, its centred values kept in e4m3."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, scale):
        v = _wide(x) * scale
        var = torch.var(v, -1, correction=0, keepdim=True)
        centred = x.float() - x.double().mean(-1, keepdim=True).float()
        ctx.save_for_backward(*_quantize(centred, "e4m3"), weight, torch.rsqrt(var + eps))
        ctx.scale, ctx.types = scale, (x.dtype, None if bias is None else bias.dtype)
        return F.layer_norm(x if scale == 1.0 else x * scale, x.shape[-1:], weight, bias, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        codes, scales, weight, r = ctx.saved_tensors
        g = _wide(grad)
        h = _dequantize(codes, scales, "e4m3", g.shape[-1], r.dtype) * ctx.scale * r
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            a = g if weight is None else g * _wide(weight)
            gx = ctx.scale * r * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
            gx = gx.to(ctx.types[0])
        if ctx.needs_input_grad[1]:
            gw = (g * h).reshape(-1, g.shape[-1]).sum(0).to(weight.dtype)
        if ctx.needs_input_grad[2]:
            gb = g.reshape(-1, g.shape[-1]).sum(0).to(ctx.types[1])
        return gx, gw, gb, None, None


def layer_norm_saved(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float, scale: float) -> Tensor:
    """The PyTorch form of a layer norm of scale * x that keeps x in e4m3."""
    return _NormSaved.apply(x, weight, bias, eps, scale)


# ---------------------------------------------------------------------------
# operators
# ---------------------------------------------------------------------------
def _autocast(*tensors: Tensor | None) -> tuple[Tensor | None, ...]:
    """The operands of a product as autocast has them where it is on."""
    kind = tensors[0].device.type
    # (asking for meta tensors raises: they have no autocast)
    if kind == "meta" or not torch.is_autocast_enabled(kind) or tensors[0].dtype == torch.float64:
        return tensors
    dtype = torch.get_autocast_dtype(kind)
    return tuple(t if t is None else t.to(dtype) for t in tensors)


def mx_quantize(x: Tensor, format: str = "e4m3", *, implementation: ImplementationMode = "native") -> MXTensor:
    """``x`` microscaled along its last axis (no gradient comes through)."""
    check_implementation(implementation)
    check_format(format)
    op = native_op("mx_quantize", x.device.type, implementation)
    if op is not None:
        try:
            return MXTensor(*op(x, format), format, x.shape[-1], x.dtype)
        except NotImplementedError:  # outside the library's limits
            if implementation == "native":
                raise
    return MXTensor(*_quantize(x, format), format, x.shape[-1], x.dtype)


def mx_dequantize(t: MXTensor, dtype: torch.dtype | None = None, *,
                  implementation: ImplementationMode = "native") -> Tensor:
    """The values of a microscaled tensor, rounded to ``dtype`` (its own by default)."""
    check_implementation(implementation)
    dtype = t.dtype if dtype is None else dtype
    op = native_op("mx_dequantize", t.device.type, implementation)
    if op is not None:
        try:
            return op(t.codes, t.scales, t.format, t.size, dtype)
        except NotImplementedError:
            if implementation == "native":
                raise
    return _dequantize(t.codes, t.scales, t.format, t.size, dtype)


def mx_linear(x: Tensor, weight: MXTensor, bias: Tensor | None = None, *, activations: str | None = None,
              implementation: ImplementationMode = "native") -> Tensor:
    """``x @ weight.T + bias`` for values ``[..., inputs]`` and an e2m1 weight
    ``[outputs, inputs]``: exact products, fp32 sums, the result in x's type.
    ``activations="e2m1"``: x is microscaled on the way in.  The weight is frozen;
    x's gradient is ``grad @ weight`` (the rounding of x passes it through)."""
    check_implementation(implementation)
    check_activations(activations)
    if weight.format != "e2m1" or weight.codes.dim() != 2:
        raise ValueError(f"mx_linear takes an e2m1 weight [outputs, inputs], got {weight.format} {tuple(weight.shape)}.")
    if x.shape[-1:] != (weight.size,):
        raise RuntimeError(f"mx_linear: a weight of shape {tuple(weight.shape)} for values of shape {tuple(x.shape)}.")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise RuntimeError(f"mx_linear: a bias of shape {tuple(bias.shape)} for {weight.shape[0]} outputs.")
    x, bias = _autocast(x, bias)
    op = native_op("mx_linear", x.device.type, implementation)
    if op is not None:
        try:
            return op(x, weight.codes, weight.scales, bias, activations)
        except NotImplementedError:
            if implementation == "native":
                raise
    return _MXLinear.apply(x, weight.codes, weight.scales, bias, activations)


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, saved: str | None = None,
           implementation: ImplementationMode = "native") -> Tensor:
    """``x @ weight.T + bias``.  ``saved="e4m3"``: x is kept in e4m3 for the weight's gradient."""
    check_implementation(implementation)
    check_saved(saved)
    if saved is None:
        return F.linear(x, weight, bias)
    x, weight, bias = _autocast(x, weight, bias)
    op = native_op("linear_saved", x.device.type, implementation)
    if op is not None:
        try:
            return op(x, weight, bias)
        except NotImplementedError:
            if implementation == "native":
                raise
    return _LinearSaved.apply(x, weight, bias)


def gelu(x: Tensor, *, saved: str | None = None, implementation: ImplementationMode = "native") -> Tensor:
    """``x * Phi(x)`` with the normal distribution function Phi.  ``saved="e4m3"``: x is
    kept in e4m3 for its gradient."""
    check_implementation(implementation)
    check_saved(saved)
    if saved is None:
        return F.gelu(x)
    op = native_op("gelu_saved", x.device.type, implementation)
    if op is not None:
        try:
            return op(x)
        except NotImplementedError:
            if implementation == "native":
                raise
    return _GELUSaved.apply(x)


# ---------------------------------------------------------------------------
# modules
# ---------------------------------------------------------------------------
class Linear(nn.Linear):
    """``nn.Linear`` (its parameters, names and initialisation) on ``linear``.  Unlike the
    function and ``LayerNorm`` it keeps its input in e4m3 unless told not to: its weight's
    gradient is that at the kept input.  ``saved=None`` gives the plain layer."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, *, saved: str | None = "e4m3",
                 implementation: ImplementationMode = "native", device=None, dtype=None) -> None:
        check_implementation(implementation)
        check_saved(saved)
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        self.saved = saved
        self.implementation = implementation

    def forward(self, x: Tensor) -> Tensor:
        return linear(x, self.weight, self.bias, saved=self.saved, implementation=self.implementation)


class GELU(nn.Module):
    """``gelu`` as a module.  Unlike the function it keeps its input in e4m3 unless told not
    to: its gradient is that at the kept input.  ``saved=None`` gives the plain activation."""

    def __init__(self, *, saved: str | None = "e4m3", implementation: ImplementationMode = "native") -> None:
        check_implementation(implementation)
        check_saved(saved)
        super().__init__()
        self.saved = saved
        self.implementation = implementation

    def forward(self, x: Tensor) -> Tensor:
        return gelu(x, saved=self.saved, implementation=self.implementation)


class MXLinear(nn.Module):
    """A linear layer with a frozen e2m1 weight (buffers ``codes`` and ``scales``), on ``mx_linear``."""

    def __init__(self, weight: MXTensor, bias: Tensor | None = None, *, activations: str | None = None,
                 implementation: ImplementationMode = "native") -> None:
        check_implementation(implementation)
        check_activations(activations)
        super().__init__()
        if weight.format != "e2m1" or weight.codes.dim() != 2:
            raise ValueError(f"MXLinear takes an e2m1 weight [outputs, inputs], got {weight.format} "
                             f"{tuple(weight.shape)}.")
        self.out_features, self.in_features = weight.shape
        self.activations = activations
        self.implementation = implementation
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_linear(cls, layer: nn.Linear, *, activations: str | None = None,
                    implementation: ImplementationMode = "native") -> MXLinear:
        """The layer with its weight rounded to e2m1."""
        weight = mx_quantize(layer.weight.detach(), "e2m1", implementation=implementation)
        return cls(weight, layer.bias, activations=activations, implementation=implementation)

    def forward(self, x: Tensor) -> Tensor:
        weight = MXTensor(self.codes, self.scales, "e2m1", self.in_features)
        bias = self.bias if self.bias is None or self.bias.dtype == x.dtype else self.bias.to(x.dtype)
        return mx_linear(x, weight, bias, activations=self.activations, implementation=self.implementation)
