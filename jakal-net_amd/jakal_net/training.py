"""The loss of a vocabulary head and the gradients' global norm.

``implementation`` as in the operators: ``"native"`` (the default here) runs the
HIP library for GPU tensors of fp32, bf16 or fp16 and raises where it cannot,
CPU tensors (and a native module without these operators) take the PyTorch form;
``"kernel"`` takes the PyTorch form where the library declines; ``"reference"``
and ``"streaming"`` are the PyTorch form.
"""

from __future__ import annotations

from typing import Iterable

import torch
from torch import Tensor
from torch.nn import functional as F

from jakal_net.core import ImplementationMode, check_implementation
from jakal_net.native_backend import native_op


def cross_entropy(logits: Tensor, target: Tensor, *, ignore_index: int = -100, reduction: str = "mean",
                  implementation: ImplementationMode = "native") -> Tensor:
    """Cross entropy of logits ``[..., classes]`` against class indices ``target [...]``.

    Half-precision logits give an fp32 loss (their gradient has their type).
    ``reduction``: "mean" over the targets that are not ``ignore_index``, "sum",
    or "none" (a loss per target, 0 where ignored).  The library gives ignored
    positions the gradient 0 whatever their logits hold, and a target outside
    the classes the loss and gradient NaN."""
    check_implementation(implementation)
    op = native_op("cross_entropy", logits.device.type, implementation)
    if op is not None:
        try:
            return op(logits, target, ignore_index, reduction)
        except NotImplementedError:  # outside the library's limits
            if implementation == "native":
                raise
    if target.shape != logits.shape[:-1]:
        raise RuntimeError(f"cross_entropy: logits of shape {tuple(logits.shape)} do not pair with targets of shape "
                           f"{tuple(target.shape)}.")
    if logits.dtype in (torch.float16, torch.bfloat16):
        logits = logits.float()
    loss = F.cross_entropy(logits.reshape(-1, logits.shape[-1]), target.reshape(-1).long(), ignore_index=ignore_index,
                           reduction=reduction)
    return loss.reshape(target.shape) if reduction == "none" else loss


def _tensors(tensors: Tensor | Iterable[Tensor | None]) -> list:
    return [tensors] if isinstance(tensors, Tensor) else list(tensors)


def _device_type(tensors: list) -> str:
    return next((t.device.type for t in tensors if t is not None), "cpu")


def _wide(t: Tensor) -> Tensor:
    return t.float() if t.dtype in (torch.float16, torch.bfloat16) else t


@torch.no_grad()
def _norm(grads: list, norm_type: float) -> Tensor:
    grads = [t for t in grads if t is not None and t.numel()]
    if not grads:
        return torch.zeros(())
    norms = torch.stack([torch.linalg.vector_norm(_wide(t), norm_type) for t in grads])
    return torch.linalg.vector_norm(norms, norm_type)


def grad_norm(grads: Tensor | Iterable[Tensor | None], norm_type: float = 2.0, *,
              implementation: ImplementationMode = "native") -> Tensor:
    """Norm over all elements of a list of tensors (None skipped), as a scalar tensor."""
    check_implementation(implementation)
    grads = _tensors(grads)
    op = native_op("grad_norm", _device_type(grads), implementation)
    if op is not None:
        try:
            return op(grads, norm_type)
        except NotImplementedError:
            if implementation == "native":
                raise
    return _norm(grads, float(norm_type))


def clip_grads(grads: Tensor | Iterable[Tensor | None], max_norm: float, norm_type: float = 2.0, *,
               out: Tensor | Iterable[Tensor | None] | None = None,
               implementation: ImplementationMode = "native") -> Tensor:
    """``grads * min(1, max_norm / (norm + 1e-6))``, in place or into ``out``
    (tensors of the same shapes, of any of the types: the fp32 gradients of
    master weights beside bf16 ones); returns the norm before clipping, as a
    scalar tensor that nothing has waited for."""
    check_implementation(implementation)
    grads = _tensors(grads)
    targets = None if out is None else _tensors(out)
    op = native_op("clip_grads", _device_type(grads), implementation)
    if op is not None:
        try:
            return op(grads, max_norm, norm_type, targets)
        except NotImplementedError:
            if implementation == "native":
                raise
    if not float(max_norm) >= 0.0:
        raise ValueError(f"clip_grads: max_norm must not be negative, got {max_norm}.")
    targets = grads if targets is None else targets
    if len(targets) != len(grads):
        raise ValueError(f"clip_grads: {len(grads)} gradients but {len(targets)} outputs.")
    norm = _norm(grads, float(norm_type))
    factor = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    with torch.no_grad():
        for g, o in zip(grads, targets):
            if g is not None:
                o.copy_(_wide(g) * factor)
    return norm


def clip_grad_norm_(parameters: Tensor | Iterable[Tensor], max_norm: float, norm_type: float = 2.0, *,
                    error_if_nonfinite: bool = False, implementation: ImplementationMode = "native") -> Tensor:
    """Clips the gradients of ``parameters`` in place to the global norm
    ``max_norm`` and returns the norm they had.  A parameter that is listed twice
    counts once.  ``error_if_nonfinite`` waits for the norm and raises before
    anything is scaled where it is not finite."""
    distinct = {id(p): p for p in _tensors(parameters)}
    grads = [p.grad for p in distinct.values() if p.grad is not None]
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type, implementation=implementation)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the total norm of order {norm_type} of the gradients is {float(norm)}, so they cannot "
                               "be clipped; error_if_nonfinite=False scales them all the same.")
    return clip_grads(grads, max_norm, norm_type, implementation=implementation)
