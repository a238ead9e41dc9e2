"""Layer norm, and the stabilisation that ends a layer update.

Every layer update of the Progressive-B model ends with ``state <- tanh(state)``
and ``val <- LayerNorm(val)`` over the scaled delta (reference
scripts/progressive_b_example.py:282-292, 1011-1024).  ``stabilize`` is that
step, scale included, as one operator; ``layer_norm`` is its norm alone.

``implementation`` as in the operators: ``"native"`` (the default here) runs the
HIP library for GPU tensors of fp32, bf16 or fp16 and raises where it cannot,
CPU tensors (and a native module without these operators) take the PyTorch form;
``"kernel"`` takes the PyTorch form where the library declines; ``"reference"``
and ``"streaming"`` are the PyTorch form.
The library computes in fp32 and rounds once; under GPU autocast half-precision
values come back in fp32, as torch's layer norm returns them there (on the CPU it
returns them in their own type, and so does the PyTorch form).

``saved="e4m3"`` keeps for the backward the centred values in 8 bits
(``jakal_net.mx``): the outputs are the same, and the gradients are the norm's
formulas with ``h = scale * r * kept``, the inverse deviation r being that of the
values themselves.
"""

from __future__ import annotations

import torch
from torch import Tensor, nn
from torch.nn import functional as F

from jakal_net.core import ImplementationMode, Layer, LayerDelta, check_implementation
from jakal_net.mx import check_saved, layer_norm_saved
from jakal_net.native_backend import native_op


def _autocast_rows(x: Tensor) -> Tensor:
    """x as an fp32 operator sees it: in fp32 where autocast is on for its device."""
    if x.dtype in (torch.bfloat16, torch.float16) and torch.is_autocast_enabled(x.device.type):
        return x.float()
    return x


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, *, eps: float = 1e-5,
               saved: str | None = None, implementation: ImplementationMode = "native") -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of ``x``."""
    check_implementation(implementation)
    check_saved(saved)
    op = native_op("layer_norm" if saved is None else "layer_norm_saved", x.device.type, implementation)
    if op is not None:
        try:
            return op(_autocast_rows(x), weight, bias, eps)
        except NotImplementedError:  # outside the library's limits
            if implementation == "native":
                raise
    if saved is not None:
        return layer_norm_saved(x, weight, bias, eps, 1.0)
    return F.layer_norm(x, x.shape[-1:], weight, bias, eps)


def stabilize(state: Tensor, val: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, *,
              eps: float = 1e-5, scale: float = 1.0, saved: str | None = None,
              implementation: ImplementationMode = "native") -> tuple[Tensor, Tensor]:
    """``(tanh(scale * state), layer_norm(scale * val))`` for states ``[..., N]`` and values ``[..., N, D]``."""
    check_implementation(implementation)
    check_saved(saved)
    op = native_op("stabilize" if saved is None else "stabilize_saved", val.device.type, implementation)
    if op is not None:
        try:
            return op(state, _autocast_rows(val), weight, bias, eps, scale)
        except NotImplementedError:
            if implementation == "native":
                raise
    if saved is not None:
        return (torch.tanh(state if scale == 1.0 else state * scale),
                layer_norm_saved(val, weight, bias, eps, scale))
    if scale != 1.0:
        state, val = state * scale, val * scale
    return torch.tanh(state), F.layer_norm(val, val.shape[-1:], weight, bias, eps)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over one axis (its parameters, names and initialisation) on ``layer_norm``."""

    saved: str | None = None

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, *,
                 saved: str | None = None, implementation: ImplementationMode = "native", device=None,
                 dtype=None) -> None:
        check_implementation(implementation)
        check_saved(saved)
        super().__init__(dim, eps, elementwise_affine, bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm takes one axis, got {self.normalized_shape}.")
        self.saved = saved
        self.implementation = implementation

    def forward(self, x: Tensor) -> Tensor:
        if x.shape[-1:] != self.normalized_shape:
            raise RuntimeError(f"LayerNorm over {self.normalized_shape[0]} elements got rows of {x.shape[-1]}.")
        return layer_norm(x, self.weight, self.bias, eps=self.eps, saved=self.saved,
                          implementation=self.implementation)


def _is_called(norm: nn.Module) -> bool:
    """Whether a norm module has to be called: another class than a layer norm, one over several axes, a forward of
    its own, or hooks on it."""
    return (type(norm) not in (LayerNorm, nn.LayerNorm) or len(norm.normalized_shape) != 1 or "forward" in vars(norm)
            or bool(norm._forward_hooks) or bool(norm._forward_pre_hooks) or bool(norm._backward_hooks)
            or bool(norm._backward_pre_hooks))


def stabilize_layer(layer: Layer, norm: nn.Module, delta: LayerDelta | None = None, scale: float = 1.0) -> Layer:
    """The layer after an update: replaced by ``scale`` times the delta, where one
    is given, then stabilised with the norm's parameters.  The path is that of
    the norm's ``implementation`` (the PyTorch form for a plain nn.LayerNorm); a
    norm of another class, or with hooks, is called on the scaled values instead."""
    state, val = (layer.state, layer.val) if delta is None else (delta.delta_state, delta.delta_val)
    if _is_called(norm):
        if scale != 1.0:
            state, val = state * scale, val * scale
        return layer.with_tensors(state=torch.tanh(state), val=norm(val))
    if val.shape[-1:] != norm.normalized_shape:
        raise RuntimeError(f"stabilize_layer: a norm over {tuple(norm.normalized_shape)} for values of width "
                           f"{val.shape[-1]}.")
    state, val = stabilize(state, val, norm.weight, norm.bias, eps=norm.eps, scale=scale,
                           saved=getattr(norm, "saved", None),
                           implementation=getattr(norm, "implementation", "streaming"))
    return layer.with_tensors(state=state, val=val)
