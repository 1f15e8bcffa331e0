"""Layer norm with its gradients, affine or modulated (one scale and shift for each sample, as the adaptive norms of a
DiT block).  No counterpart in the reference; the norm that feeds a quantized linear without gradients is
``ConvRotLinear.forward_modulated_norm``."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .core import _dtype_code, _require_cuda


def _address(t):
    return None if t is None else t.data_ptr()


def _forward(x, weight, bias, segments, add_one, eps, stats):
    """weight and bias: vectors that follow one another at the same stride, one for each segment of the rows."""

    features = x.shape[-1]
    rows = x.numel() // features
    y = torch.empty_like(x)
    vector = weight if weight is not None else bias
    saved = torch.empty((2, rows), dtype=torch.float32, device=x.device) if stats else None
    mean = saved.data_ptr() if stats and rows else None
    _lib.call("convrot_layer_norm", x.get_device(), x.data_ptr(), _dtype_code(x.dtype), rows, features,
              _address(weight), _address(bias), _dtype_code(x.dtype if vector is None else vector.dtype),
              max(1, rows // segments), features if segments == 1 else vector.stride(0), add_one, eps, y.data_ptr(), mean,
              None if mean is None else mean + 4 * rows)
    return y, saved


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, segments, add_one, eps):
        y, saved = _forward(x, weight, bias, segments, add_one, eps, True)
        ctx.save_for_backward(x, weight, saved)
        ctx.how = (segments, add_one, None if bias is None else (bias.shape, bias.dtype))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, saved = ctx.saved_tensors
        segments, add_one, bias = ctx.how
        _, want_w, want_b, *_ = ctx.needs_input_grad
        dy = dy.contiguous()
        features = x.shape[-1]
        rows = x.numel() // features
        per = max(1, rows // segments)
        dx = torch.empty_like(x)
        make = torch.empty if rows else torch.zeros
        dw = make(weight.shape, dtype=weight.dtype, device=x.device) if want_w else None
        db = make(bias[0], dtype=bias[1], device=x.device) if want_b else None
        size, space = 0, None
        if want_w or want_b:
            size = _lib.load().convrot_layer_norm_workspace(rows, features, per)
            space = torch.empty((size,), dtype=torch.uint8, device=x.device)
        sums_dtype = weight.dtype if weight is not None else bias[1] if bias is not None else x.dtype
        mean = saved.data_ptr()
        _lib.call("convrot_layer_norm_backward", x.get_device(), x.data_ptr(), dy.data_ptr(), _dtype_code(x.dtype), rows,
                  features, _address(weight), _dtype_code(sums_dtype), per,
                  features if weight is None or segments == 1 else weight.stride(0), add_one, mean, mean + 4 * rows,
                  dx.data_ptr(), _address(dw), _address(db), _address(space), size)
        return dx, dw, db, None, None, None


def _run(x, weight, bias, segments, add_one, eps):
    if eps < 0:
        raise ValueError(f"eps must be non-negative, got {eps}")
    _dtype_code(x.dtype)
    _require_cuda(x, weight, bias)
    types = {v.dtype for v in (weight, bias) if v is not None}
    if types not in (set(), {x.dtype}, {torch.float32}):
        weight, bias = (None if v is None else v.float() for v in (weight, bias))
    if not x.is_contiguous():
        x = x.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, segments, add_one, float(eps))
    return _forward(x, weight, bias, segments, add_one, float(eps), False)[0]


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
    if weight is not None and weight.stride(0) != 1:
        weight = weight.contiguous()
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    return _run(x, weight, bias, 1, False, eps)


def modulated_layer_norm(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``layer_norm(x) * (1 + scale) + shift`` with one scale and shift for each sample, in float32, rounded once.

    x: (batch, ..., features); shift and scale: (batch, 1, features) or
    (batch, features), columns of a wider modulation output included; a batch
    of 1 is shared by all samples.  Differentiable in all three; the gradients
    of scale and shift are float32 sums over their sample's rows."""

    if x.ndim < 2 or x.shape[-1] == 0:
        raise ValueError(f"modulated layer norm expects (batch, ..., features), got {tuple(x.shape)}")
    batch, features = x.shape[0], x.shape[-1]
    for v in (shift, scale):
        if v.shape not in ((batch, 1, features), (batch, features), (1, 1, features), (1, features)):
            raise ValueError(f"modulation vector of shape {tuple(v.shape)} does not match ({batch}, 1, {features})")
    if shift.shape[0] != scale.shape[0]:  # the shared one is repeated, its gradient summed over the samples
        shift, scale = (v.reshape(-1, features).expand(batch, features) for v in (shift, scale))
    if (shift.stride(-1) != 1 or scale.stride(-1) != 1
            or (scale.shape[0] > 1 and (shift.stride(0) != scale.stride(0) or scale.stride(0) < features))):
        shift, scale = shift.contiguous(), scale.contiguous()
    return _run(x, scale, shift, max(1, scale.shape[0]), True, eps)
