"""The 8-bit linear: int8 weights with one scale for each channel, activations
quantized to int8 with one scale for each token on the way in, an exact int32
product on the tensor cores.

For the layers of a quantized model that 4 bits hurt, and for fine-tuning
around frozen weights: the output is differentiable in the activation, whose
gradient is the same 8-bit product with the weight contracted over its other
dimension.  No counterpart in the reference (its linears are 4-bit,
src/convrot_mlx/core.py:1210-1313, and have no gradient).
"""

from __future__ import annotations

import torch
from torch import nn

from . import _lib, _native
from .core import _dtype_code, _f32_vec, _require_cuda

INT8_MAX = 127
_PITCH = 16  # rows of codes start on multiples of 16 bytes


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as (rows, features) with unit stride along the features and rows that do not overlap."""

    x2 = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1 or x2.stride(0) < x2.shape[1]:
        x2 = x2.contiguous()
        if x2.stride(0) < x2.shape[1]:  # a single row of a stride that was never needed
            x2 = x2.as_strided(x2.shape, (x2.shape[1], 1))
    return x2


def _f32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.float32 and t.is_contiguous() else _f32_vec(t)


def _padded_rows(codes: torch.Tensor) -> torch.Tensor:
    """int8 rows on a pitch of a multiple of 16 bytes (a copy only when they are not)."""

    if codes.stride(1) == 1 and codes.stride(0) >= codes.shape[1] and codes.stride(0) % _PITCH == 0 \
            and codes.data_ptr() % _PITCH == 0:
        return codes
    rows, features = codes.shape
    out = torch.empty((rows, -(-features // _PITCH) * _PITCH), dtype=torch.int8, device=codes.device)[:, :features]
    return out.copy_(codes)


def _quantize(x2: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    rows, features = x2.shape
    codes = torch.empty((rows, -(-features // _PITCH) * _PITCH), dtype=torch.int8, device=x2.device)
    scales = torch.empty((rows,), dtype=torch.float32, device=x2.device)
    _lib.call("convrot_quantize_i8", x2.get_device(), x2.data_ptr(), _dtype_code(x2.dtype), rows, features,
              x2.stride(0), None, codes.data_ptr(), codes.shape[1], scales.data_ptr())
    return codes[:, :features], scales


def quantize_signed_int8_rowwise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Symmetric 8-bit quantization of each row: codes in [-127, 127] and float32 scales (absmax / 127).

    The codes come on rows padded to a multiple of 16 bytes (a view of them),
    as ``int8_matmul`` reads them.  A zero row has codes and scale 0; a row
    with an infinity or a NaN has codes 0 and scale NaN."""

    if x.ndim != 2 or x.shape[1] == 0:
        raise ValueError(f"rowwise int8 quantization expects 2D input with features, got {tuple(x.shape)}")
    _require_cuda(x)
    return _quantize(_rows(x))


def quantize_int8_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (out, in) and channel scales (out,) of a dense (out, in) weight."""

    if weight.ndim != 2:
        raise ValueError(f"int8 weight must be 2D, got {tuple(weight.shape)}")
    return quantize_signed_int8_rowwise(weight)


def _validate(k: int, qweight, wscales, bias) -> int:
    if qweight.ndim != 2 or qweight.dtype != torch.int8:
        raise ValueError(f"int8 weight must be a 2D int8 tensor, got {tuple(qweight.shape)} {qweight.dtype}")
    n = qweight.shape[0]
    if qweight.shape[1] != k or k == 0:
        raise ValueError(f"int8 weight must be (N, K) rows; activation K={k}, weight={tuple(qweight.shape)}")
    if tuple(wscales.shape) != (n,):
        raise ValueError(f"int8 weight scales must have shape {(n,)}, got {tuple(wscales.shape)}")
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"int8 bias must have shape {(n,)}, got {tuple(bias.shape)}")
    return n


def int8_matmul(codes, qweight, xscales, wscales, bias=None, *, output_dtype) -> torch.Tensor:
    """``output_dtype(float(codes @ qweight.T) * xscales * wscales + bias)`` with an exact int32 dot.

    codes: (m, k) int8 and xscales (m,), as ``quantize_signed_int8_rowwise``
    gives them; qweight: (n, k) int8 with wscales (n,).  Rows that do not
    start on multiples of 16 bytes are copied first."""

    if codes.ndim != 2 or codes.dtype != torch.int8:
        raise ValueError(f"int8 product requires a 2D int8 activation, got {tuple(codes.shape)} {codes.dtype}")
    n = _validate(codes.shape[1], qweight, wscales, bias)
    if tuple(xscales.shape) != (codes.shape[0],):
        raise ValueError(f"int8 activation scales must have shape {(codes.shape[0],)}, got {tuple(xscales.shape)}")
    _dtype_code(output_dtype)
    _require_cuda(codes, qweight, xscales, wscales, bias)
    for t in (qweight, xscales, wscales, bias):
        if t is not None and t.device != codes.device:
            raise ValueError(f"expected all tensors on {codes.device}, got one on {t.device}")
    codes, qweight, xscales, wscales = _padded_rows(codes), _padded_rows(qweight), _f32(xscales), _f32(wscales)
    bias = None if bias is None else _f32(bias)
    m, k = codes.shape
    out = torch.empty((m, n), dtype=output_dtype, device=codes.device)
    _lib.call("convrot_i8_gemm", codes.get_device(), codes.data_ptr(), codes.stride(0), qweight.data_ptr(),
              qweight.stride(0), _lib.LAYOUT_NK, xscales.data_ptr(), wscales.data_ptr(),
              None if bias is None else bias.data_ptr(), out.data_ptr(), _dtype_code(output_dtype), m, n, k)
    return out


def int8_linear(x: torch.Tensor, qweight: torch.Tensor, wscales: torch.Tensor,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ (qweight * wscales[:, None]).T + bias`` with x quantized to 8 bits for each token.

    x: (..., k) float32, float16 or bfloat16; qweight: (n, k) int8, best on
    rows padded to 16 bytes as ``quantize_int8_weight`` returns it (else every
    call copies it); wscales, bias: (n,).  Differentiable in x: the gradient
    dy * wscales is quantized for each token in turn and multiplied with the
    same weight.  The weight, its scales and the bias are frozen.

    k is at most 131072, what an exact int32 dot can sum; of more than 131072
    channels n the gradient adds the exact dots of ranges in float32."""

    return _native.ops().int8_linear(x, qweight, wscales, bias)


class Int8Linear(nn.Module):
    """A frozen linear layer held in 8 bits (``int8_linear``).  ``qweight`` keeps the codes on rows padded to 16
    bytes; ``scales`` and ``bias`` are float32 buffers, and stay so when the module is cast to another type."""

    def __init__(self, in_features: int, out_features: int, *, bias: bool = True, device=None):
        super().__init__()
        if in_features < 1 or out_features < 1:
            raise ValueError(f"Int8Linear needs positive sizes, got {in_features} x {out_features}")
        self.in_features = in_features
        self.out_features = out_features
        pitch = -(-in_features // _PITCH) * _PITCH
        self.register_buffer("qweight", torch.zeros((out_features, pitch), dtype=torch.int8, device=device))
        self.register_buffer("scales", torch.ones((out_features,), dtype=torch.float32, device=device))
        self.register_buffer("bias", torch.zeros((out_features,), dtype=torch.float32, device=device) if bias else None)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Linear) -> "Int8Linear":
        """The 8-bit form of a dense layer on a CUDA device."""

        layer = cls(linear.in_features, linear.out_features, bias=linear.bias is not None, device=linear.weight.device)
        codes, scales = quantize_int8_weight(linear.weight.detach())
        layer.qweight[:, :linear.in_features] = codes
        layer.scales = scales
        if linear.bias is not None:
            layer.bias = linear.bias.detach().float().clone()
        return layer

    def _apply(self, fn, *args, **kwargs):
        # a cast would round each channel's scale (by up to 2^-9 in bfloat16): only the device follows it
        held = {name: self._buffers[name] for name in ("scales", "bias") if self._buffers[name] is not None}
        super()._apply(fn, *args, **kwargs)
        for name, value in held.items():
            cast = self._buffers[name]
            if cast.dtype != torch.float32:
                self._buffers[name] = value.to(device=cast.device, dtype=torch.float32)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Int8Linear expected K={self.in_features}, got {x.shape[-1]}")
        return int8_linear(x, self.qweight[:, :self.in_features], self.scales, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
