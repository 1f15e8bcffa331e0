"""Activations of a training step whose saved input is held in 8 bits.  No counterpart in the reference."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .core import _dtype_code, _require_cuda

SAVED_GROUP = 128  # features of a row that share one scale


def _forward(x, save: bool):
    features = x.shape[-1]
    rows = x.numel() // features
    y = torch.empty_like(x)
    codes = scales = None
    if save:
        codes = torch.empty((rows, features), dtype=torch.int8, device=x.device)
        scales = torch.empty((rows, -(-features // SAVED_GROUP)), dtype=torch.float32, device=x.device)
    _lib.call("convrot_gelu_saved8", x.get_device(), x.data_ptr(), _dtype_code(x.dtype), rows, features, y.data_ptr(),
              codes.data_ptr() if save else None, scales.data_ptr() if save else None)
    return y, codes, scales


class _GeluSaved8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y, codes, scales = _forward(x, True)
        ctx.save_for_backward(codes, scales)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales = ctx.saved_tensors
        dy = dy.contiguous()
        dx = torch.empty_like(dy)
        _lib.call("convrot_gelu_saved8_backward", dy.get_device(), dy.data_ptr(), _dtype_code(dy.dtype), codes.shape[0],
                  codes.shape[1], codes.data_ptr(), scales.data_ptr(), dx.data_ptr())
        return dx


def gelu_tanh_saved8(x: torch.Tensor) -> torch.Tensor:
    """Tanh GELU whose backward pass reads its input from 8 bits.

    The output is that of the input as given; for the backward pass only int8
    codes of x are kept, with one float32 scale for each 128 features of a
    row: about half of a 16-bit x, and none of x itself.  The gradient is the
    formula's at the restored input, at most half a code step (1/254 of its
    group's largest magnitude) away."""

    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError(f"gelu expects features in the last dimension, got {tuple(x.shape)}")
    _dtype_code(x.dtype)
    _require_cuda(x)
    x = x.contiguous()
    if torch.is_grad_enabled() and x.requires_grad:
        return _GeluSaved8.apply(x)
    return _forward(x, False)[0]
