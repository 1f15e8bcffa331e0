"""Layer norm with its gradients, affine or modulated (one scale and shift for each sample, as the adaptive norms of a
DiT block).  No counterpart in the reference; the norm that feeds a quantized linear without gradients is
``ConvRotLinear.forward_modulated_norm``."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .core import _dtype_code, _require_cuda


def _forward(x, weight, bias, rows_per_weight, add_one, eps, stats):
    features = x.shape[-1]
    rows = x.numel() // features
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean, rstd = torch.empty((2, rows), dtype=torch.float32, device=x.device) if stats else (None, None)
    vector = weight if weight is not None else bias
    _lib.call("convrot_layer_norm", x, _lib.ptr(x), _dtype_code(x.dtype), rows, features, _lib.ptr(weight),
              _lib.ptr(bias), _dtype_code(x.dtype if vector is None else vector.dtype), rows_per_weight,
              features if vector is None else vector.stride(0), int(add_one), eps, _lib.ptr(y), _lib.ptr(mean),
              _lib.ptr(rstd))
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    """weight and bias: None or (segments, features) of one dtype and stride."""

    @staticmethod
    def forward(ctx, x, weight, bias, rows_per_weight, add_one, eps):
        y, mean, rstd = _forward(x, weight, bias, rows_per_weight, add_one, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.how = (rows_per_weight, add_one, None if bias is None else (bias.shape, bias.dtype))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        rows_per_weight, add_one, bias = ctx.how
        _, want_w, want_b = ctx.needs_input_grad[:3]
        dy = dy.contiguous()
        features = x.shape[-1]
        rows = x.numel() // features
        dx = torch.empty_like(x)
        make = torch.empty if rows else torch.zeros
        dw = make(weight.shape, dtype=weight.dtype, device=x.device) if want_w else None
        db = make(bias[0], dtype=bias[1], device=x.device) if want_b else None
        size = _lib.load().convrot_layer_norm_workspace(rows, features, rows_per_weight) if want_w or want_b else 0
        space = torch.empty((size,), dtype=torch.uint8, device=x.device) if size else None
        sums_dtype = weight.dtype if weight is not None else bias[1] if bias is not None else x.dtype
        _lib.call("convrot_layer_norm_backward", x, _lib.ptr(x), _lib.ptr(dy), _dtype_code(x.dtype), rows, features,
                  _lib.ptr(weight), _dtype_code(sums_dtype), rows_per_weight,
                  features if weight is None else weight.stride(0), int(add_one), _lib.ptr(mean), _lib.ptr(rstd),
                  _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(space), size)
        return dx, dw, db, None, None, None


def _vectors(x, weight, bias):
    """Both vectors as (segments, features) of one stride and of x's dtype, or both float32."""

    given = [v for v in (weight, bias) if v is not None]
    if any(v.dtype != given[0].dtype for v in given) or (given and given[0].dtype not in (x.dtype, torch.float32)):
        weight, bias = (None if v is None else v.float() for v in (weight, bias))
    given = [v for v in (weight, bias) if v is not None]
    if any(v.stride(1) != 1 or v.stride(0) < v.shape[1] or v.stride(0) != given[0].stride(0) for v in given):
        weight, bias = (None if v is None else v.contiguous() for v in (weight, bias))
    return weight, bias


def _run(x, weight, bias, rows_per_weight, add_one, eps):
    if eps < 0:
        raise ValueError(f"eps must be non-negative, got {eps}")
    _dtype_code(x.dtype)
    _require_cuda(x, weight, bias)
    weight, bias = _vectors(x, weight, bias)
    x = x.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, rows_per_weight, add_one, float(eps))
    return _forward(x, weight, bias, rows_per_weight, add_one, float(eps), False)[0]


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in float32, rounded once.

    x: (..., features) float32, float16 or bfloat16; weight and bias:
    (features,) or None.  Differentiable in all three; the gradients of weight
    and bias are float32 sums over all rows, in an order that depends on the
    shape alone."""

    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer norm expects features in the last dimension, got {tuple(x.shape)}")
    features = x.shape[-1]
    for v, name in ((weight, "weight"), (bias, "bias")):
        if v is not None and tuple(v.shape) != (features,):
            raise ValueError(f"layer norm {name} must have shape {(features,)}, got {tuple(v.shape)}")
    weight, bias = (None if v is None else v.unsqueeze(0) for v in (weight, bias))
    return _run(x, weight, bias, max(1, x.numel() // features), False, eps)


def modulated_layer_norm(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``layer_norm(x) * (1 + scale) + shift`` with one scale and shift for each sample, in float32, rounded once.

    x: (batch, ..., features); shift and scale: (batch, 1, features) or
    (batch, features), columns of a wider modulation output included; a batch
    of 1 is shared by all samples.  Differentiable in all three; the gradients
    of scale and shift are float32 sums over their sample's rows."""

    if x.ndim < 2 or x.shape[-1] == 0:
        raise ValueError(f"modulated layer norm expects (batch, ..., features), got {tuple(x.shape)}")
    batch, features = x.shape[0], x.shape[-1]
    vectors = []
    for v in (shift, scale):
        v2 = v[:, 0] if v.ndim == 3 and v.shape[1] == 1 else v
        if v2.ndim != 2 or v2.shape[1] != features or v2.shape[0] not in (1, batch):
            raise ValueError(f"modulation vector of shape {tuple(v.shape)} does not match ({batch}, 1, {features})")
        vectors.append(v2)
    shift, scale = vectors
    segments = max(shift.shape[0], scale.shape[0])
    if shift.shape[0] != scale.shape[0]:  # the shared one is repeated, its gradient summed over the samples
        shift, scale = shift.expand(segments, features).contiguous(), scale.expand(segments, features).contiguous()
    rows = x.numel() // features
    return _run(x, scale, shift, max(1, rows // max(1, segments)), True, eps)
