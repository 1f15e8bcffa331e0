"""The 8-bit floating-point linear: e4m3 weights with one power-of-two scale for
each block of 128 x 128, activations quantized on the way in with one for each
128 values of a token, and a product on the tensor cores that applies the
scales itself.

It stands beside the 8-bit integer linear (``int8_linear``) for the layers that
4 bits hurt: there a token has one scale, so a channel twenty times larger
than the others costs all of them four of their bits, here it costs those of its
block at most.  Frozen weights; the output is differentiable in the activation,
whose gradient is the same product with the weight contracted over its other
dimension.  No counterpart in the reference (its linears are 4-bit,
src/convrot_mlx/core.py:1210-1313, and have no gradient).
"""

from __future__ import annotations

import torch
from torch import nn

from . import _lib, _native
from .core import _dtype_code, _require_cuda
from .int8 import _PITCH, _f32, _rows

FP8_SPAN = 128  # values of a row, rows and columns of a weight, that share a scale
CODES = torch.float8_e4m3fn
SCALES = torch.float8_e8m0fnu


def _spans(n: int) -> int:
    return -(-n // FP8_SPAN)


def _padded_codes(codes: torch.Tensor) -> torch.Tensor:
    """Rows of codes on a pitch of a multiple of 16 bytes, the last one's padding too (a copy only when they are not)."""

    rows, features = codes.shape
    if codes.stride(1) == 1 and codes.stride(0) >= features and codes.stride(0) % _PITCH == 0 \
            and codes.data_ptr() % _PITCH == 0 and codes.untyped_storage().nbytes() >= \
            codes.storage_offset() + (rows - 1) * codes.stride(0) + -(-features // _PITCH) * _PITCH:
        return codes
    out = torch.empty((rows, -(-features // _PITCH) * _PITCH), dtype=codes.dtype, device=codes.device)[:, :features]
    return out.copy_(codes)


def _padded_scales(scales: torch.Tensor) -> torch.Tensor:
    """Rows of scales at multiples of 4 bytes that pad them to such a multiple."""

    rows, spans = scales.shape
    pitch = -(-spans // 4) * 4
    if scales.stride(1) == 1 and scales.stride(0) >= pitch and scales.stride(0) % 4 == 0 and scales.data_ptr() % 4 == 0 \
            and scales.untyped_storage().nbytes() >= scales.storage_offset() + (rows - 1) * scales.stride(0) + pitch:
        return scales
    out = torch.zeros((rows, pitch), dtype=torch.uint8, device=scales.device)
    out[:, :spans] = scales.view(torch.uint8)
    return out.view(SCALES)[:, :spans]


def _check_2d(x: torch.Tensor, what: str) -> None:
    if x.ndim != 2 or x.shape[1] == 0:
        raise ValueError(f"{what} expects 2D input with features, got {tuple(x.shape)}")
    _dtype_code(x.dtype)
    _require_cuda(x)


def quantize_fp8_blockwise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes of the rows of x and one power-of-two scale (float8_e8m0fnu) for each 128 values of a row.

    The scale is the least 2^e, e >= -127, with max|x| <= 448 * 2^e in the block, so
    codes are rounded once, to nearest even.  Codes (rows, features) and scales
    (rows, ceil(features / 128)) come on padded rows (views of them), as
    ``fp8_matmul`` reads them.  A block that holds an infinity or a NaN has codes 0
    and scale NaN."""

    _check_2d(x, "blockwise fp8 quantization")
    x = _rows(x.detach())
    rows, features = x.shape
    codes = torch.empty((rows, -(-features // _PITCH) * _PITCH), dtype=CODES, device=x.device)
    scales = torch.empty((rows, -(-_spans(features) // 4) * 4), dtype=SCALES, device=x.device)
    _lib.call("convrot_quantize_fp8", x.get_device(), x.data_ptr(), _dtype_code(x.dtype), rows, features, x.stride(0),
              codes.data_ptr(), codes.shape[1], scales.data_ptr(), scales.shape[1])
    return codes[:, :features], scales[:, :_spans(features)]


def quantize_fp8_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes (out, in), on rows padded to 16 bytes, and the power-of-two scales (ceil(out / 128), ceil(in / 128))
    of a dense (out, in) weight's blocks of 128 x 128."""

    _check_2d(weight, "fp8 weight quantization")
    w = _rows(weight.detach())
    n, k = w.shape
    codes = torch.empty((n, -(-k // _PITCH) * _PITCH), dtype=CODES, device=w.device)
    scales = torch.empty((_spans(n), _spans(k)), dtype=SCALES, device=w.device)
    _lib.call("convrot_quantize_fp8_weight", w.get_device(), w.data_ptr(), _dtype_code(w.dtype), n, k, w.stride(0),
              codes.data_ptr(), codes.shape[1], scales.data_ptr(), _spans(k))
    return codes[:, :k], scales


def fp8_matmul(codes, qweight, xscales, wscales, bias=None, *, output_dtype) -> torch.Tensor:
    """The product of ``codes`` (m, k) and ``qweight`` (n, k) transposed, each code times its block's scale, plus bias.

    Arguments as ``quantize_fp8_blockwise`` and ``quantize_fp8_weight`` give
    them; sums are float32, rounded once to ``output_dtype`` (float32 outputs over more
    than 8192 channels are summed in ranges).  Rows that do not start where the kernel can
    read them are copied first.  No gradients: ``fp8_linear`` has them."""

    for t, what in ((codes, "activation"), (qweight, "weight")):
        if t.ndim != 2 or t.dtype != CODES:
            raise ValueError(f"fp8 product requires a 2D float8_e4m3fn {what}, got {tuple(t.shape)} {t.dtype}")
    (m, k), n = codes.shape, qweight.shape[0]
    if qweight.shape[1] != k or k == 0 or n == 0:
        raise ValueError(f"fp8 weight must be (N, K) rows; activation K={k}, weight={tuple(qweight.shape)}")
    for t, want, what in ((xscales, (m, _spans(k)), "activation"), (wscales, (_spans(n), _spans(k)), "weight")):
        if tuple(t.shape) != want or t.dtype != SCALES:
            raise ValueError(f"fp8 {what} scales must be {want} float8_e8m0fnu, got {tuple(t.shape)} {t.dtype}")
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"fp8 bias must have shape {(n,)}, got {tuple(bias.shape)}")
    _dtype_code(output_dtype)
    _require_cuda(codes, qweight, xscales, wscales, bias)
    for t in (qweight, xscales, wscales, bias):
        if t is not None and t.device != codes.device:
            raise ValueError(f"expected all tensors on {codes.device}, got one on {t.device}")
    out = torch.empty((m, n), dtype=output_dtype, device=codes.device)
    if m == 0:
        return out
    codes, qweight, xscales, wscales = _padded_codes(codes), _padded_codes(qweight), _padded_scales(xscales), wscales.contiguous()
    bias = None if bias is None else _f32(bias)
    _lib.call("convrot_fp8_gemm", codes.get_device(), codes.data_ptr(), codes.stride(0), xscales.data_ptr(), xscales.stride(0),
              qweight.data_ptr(), qweight.stride(0), _lib.LAYOUT_NK, wscales.data_ptr(), _spans(k),
              None if bias is None else bias.data_ptr(), out.data_ptr(), _dtype_code(output_dtype), m, n, k)
    return out


def fp8_linear(x: torch.Tensor, qweight: torch.Tensor, wscales: torch.Tensor,
               bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` with x quantized to e4m3 with a power-of-two scale for each 128 values of a token.

    x: (..., k) float32, float16 or bfloat16; W: ``qweight`` (n, k)
    float8_e4m3fn times ``wscales`` (ceil(n / 128), ceil(k / 128)) float8_e8m0fnu
    for its blocks, as ``quantize_fp8_weight`` returns them (rows that are not on
    a multiple of 16 bytes are copied by every call); bias: (n,).
    Differentiable in x: the gradient dy is quantized in the same way along its
    channels and multiplied with the same weight.  The weight, its scales and the
    bias are frozen.  A token with an infinity or a NaN has outputs NaN."""

    return _native.ops().fp8_linear(x, qweight, wscales, bias)


class Fp8Linear(nn.Module):
    """A frozen linear layer held in 8-bit floating point (``fp8_linear``).  ``qweight`` keeps the codes as bytes on rows
    padded to 16, ``scales`` the exponents' bytes, so that casts of the module leave both alone; ``bias`` is a float32
    buffer, and stays so."""

    def __init__(self, in_features: int, out_features: int, *, bias: bool = True, device=None):
        super().__init__()
        if in_features < 1 or out_features < 1:
            raise ValueError(f"Fp8Linear needs positive sizes, got {in_features} x {out_features}")
        self.in_features = in_features
        self.out_features = out_features
        pitch = -(-in_features // _PITCH) * _PITCH
        self.register_buffer("qweight", torch.zeros((out_features, pitch), dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.full((_spans(out_features), _spans(in_features)), 127, dtype=torch.uint8,
                                                  device=device))
        self.register_buffer("bias", torch.zeros((out_features,), dtype=torch.float32, device=device) if bias else None)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Linear) -> "Fp8Linear":
        """The 8-bit form of a dense layer on a CUDA device."""

        layer = cls(linear.in_features, linear.out_features, bias=linear.bias is not None, device=linear.weight.device)
        codes, scales = quantize_fp8_weight(linear.weight)
        layer.qweight[:, :linear.in_features] = codes.view(torch.uint8)
        layer.scales = scales.view(torch.uint8)
        if linear.bias is not None:
            layer.bias = linear.bias.detach().float().clone()
        return layer

    def _apply(self, fn, *args, **kwargs):
        # a cast would round the bias: only the device follows it
        held = self._buffers["bias"]
        super()._apply(fn, *args, **kwargs)
        if held is not None and self._buffers["bias"].dtype != torch.float32:
            self._buffers["bias"] = held.to(device=self._buffers["bias"].device, dtype=torch.float32)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Fp8Linear expected K={self.in_features}, got {x.shape[-1]}")
        return fp8_linear(x, self.qweight.view(CODES)[:, :self.in_features], self.scales.view(SCALES), self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
