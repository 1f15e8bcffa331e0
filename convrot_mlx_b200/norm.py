"""Layer norm with its gradients, affine or modulated (one scale and shift for each sample, as the adaptive norms of a
DiT block).  No counterpart in the reference; the norm that feeds a quantized linear without gradients is
``ConvRotLinear.forward_modulated_norm``."""

from __future__ import annotations

import torch

from . import _native


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in float32, rounded once.

    x: (..., features) float32, float16 or bfloat16; weight and bias:
    (features,) or None.  Differentiable in all three; the gradients of weight
    and bias are float32 sums over all rows, in an order that depends on the
    shape, the types, the tensors' alignment and the GPU's size, but not from
    run to run."""

    return _native.ops().layer_norm(x, weight, bias, eps)


def modulated_layer_norm(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``layer_norm(x) * (1 + scale) + shift`` with one scale and shift for each sample, in float32, rounded once.

    x: (batch, ..., features); shift and scale: (batch, 1, features) or
    (batch, features), columns of a wider modulation output included; a batch
    of 1 is shared by all samples.  At most 65535 samples may have a shift and
    scale of their own.  Differentiable in all three; the gradients of scale and
    shift are float32 sums over their sample's rows, ordered as in
    ``layer_norm``."""

    return _native.ops().modulated_layer_norm(x, shift, scale, eps)
