"""Jakal-Net operator API, MI355X build of the native hot path.

Public names of the reference's ``src/jakal_net/__init__.py:1-70`` that belong
to the hot path: layers, the propagation / transition operators, the low-rank
score modules and the native-backend status calls; beside them the operators of
a training step (layer norm and the layer update's stabilisation, the vocabulary
loss, and the gradients' norm) and those on microscaled numbers: layers that keep
their inputs in 8 bits for the backward, products by 4-bit weights.
"""

from jakal_net.core import Layer, LayerDelta
from jakal_net.modules import (
    LowRankBilinearPairwise,
    LowRankBilinearRoute,
    MultiHeadPairwise,
    MultiHeadRoute,
    TemperatureScaledRoute,
)
from jakal_net.mx import GELU, Linear, MXLinear, MXTensor, gelu, linear, mx_dequantize, mx_linear, mx_quantize
from jakal_net.native_backend import native_available, native_status
from jakal_net.norm import LayerNorm, layer_norm, stabilize, stabilize_layer
from jakal_net.propagation import Propagation, SparsePropagation
from jakal_net.training import clip_grad_norm_, clip_grads, cross_entropy, grad_norm
from jakal_net.transition import SparseTransition, Transition

__all__ = [
    "GELU",
    "Layer",
    "LayerDelta",
    "LayerNorm",
    "Linear",
    "LowRankBilinearPairwise",
    "LowRankBilinearRoute",
    "MXLinear",
    "MXTensor",
    "MultiHeadPairwise",
    "MultiHeadRoute",
    "Propagation",
    "SparsePropagation",
    "SparseTransition",
    "TemperatureScaledRoute",
    "Transition",
    "clip_grad_norm_",
    "clip_grads",
    "cross_entropy",
    "gelu",
    "grad_norm",
    "layer_norm",
    "linear",
    "mx_dequantize",
    "mx_linear",
    "mx_quantize",
    "native_available",
    "native_status",
    "stabilize",
    "stabilize_layer",
]
