"""Host-side checks of the 8-bit floating-point linear (no GPU needed): refusals before any device work, and the shapes
that make no work."""

from __future__ import annotations

import ctypes

import pytest
import torch

import convrot_mlx_b200 as cr
from convrot_mlx_b200 import _lib

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below ends in its checks


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _err(lib):
    return lib.convrot_last_error().decode()


@pytest.mark.parametrize("name", ["convrot_quantize_fp8", "convrot_quantize_fp8_weight"])
def test_fp8_quantizer_arguments(lib, name):
    def run(dtype=2, rows=4, features=300, stride=300, pitch=304, scales_pitch=4, x=FAKE, codes=FAKE, scales=FAKE):
        return getattr(lib, name)(x, dtype, rows, features, stride, codes, pitch, scales, scales_pitch, None)

    assert run(dtype=7) == -1 and "dtype" in _err(lib)
    assert run(rows=-1) == -1 and run(features=0) == -1
    assert run(stride=299) == -1 and "strides" in _err(lib)
    assert run(pitch=288) == -1 and run(pitch=300) == -1 and run(scales_pitch=2) == -1
    assert run(x=None) == -1 and run(codes=None) == -1 and run(scales=None) == -1
    assert run(codes=ctypes.c_void_p(4104)) == -1 and "aligned" in _err(lib)
    assert run(x=ctypes.c_void_p(4097)) == -1
    assert run(rows=1 << 30) == -2
    assert run(rows=0) == 0


def _gemm(lib, m=4, n=300, k=400, sa=400, sw=400, layout=0, dtype=2, xs=4, ws=4, act=FAKE, weight=FAKE, out=FAKE,
          xscales=FAKE, wscales=FAKE):
    return lib.convrot_fp8_gemm(act, sa, xscales, xs, weight, sw, layout, wscales, ws, None, out, dtype, m, n, k, None)


def test_fp8_gemm_arguments(lib):
    assert _gemm(lib, layout=2) == -1 and _gemm(lib, dtype=5) == -1
    assert _gemm(lib, m=-1) == -1 and _gemm(lib, n=0) == -1 and _gemm(lib, k=0) == -1
    assert _gemm(lib, sa=384) == -1 and _gemm(lib, sw=408) == -1 and "multiples of 16" in _err(lib)
    assert _gemm(lib, layout=1, sw=288) == -1  # (k, n) rows do not cover n
    assert _gemm(lib, xs=3) == -1 and _gemm(lib, xs=6) == -1 and _gemm(lib, ws=3) == -1 and "scales" in _err(lib)
    assert _gemm(lib, layout=1, sw=304, ws=2) == -1
    assert _gemm(lib, n=1 << 22) == -2
    assert _gemm(lib, act=ctypes.c_void_p(4098)) == -1 and "aligned" in _err(lib)
    assert _gemm(lib, xscales=ctypes.c_void_p(4098)) == -1
    for name in ("act", "weight", "out", "xscales", "wscales"):
        assert _gemm(lib, **{name: None}) == -1
    assert _gemm(lib, m=0) == 0


def test_fp8_linear_arguments(lib):
    def run(dtype=2, m=4, k=400, pitch=400, codes=FAKE, x=FAKE, stride=400, scales_pitch=4):
        return lib.convrot_fp8_linear(x, dtype, stride, FAKE, 400, 0, FAKE, 4, None, FAKE, dtype, m, 300, k, codes, pitch,
                                      FAKE, scales_pitch, None)

    assert run(dtype=3) == -1 and run(pitch=392) == -1 and run(codes=None) == -1 and run(scales_pitch=2) == -1
    assert run(x=None) == -1 and run(stride=399) == -1
    assert run(m=0) == 0


def test_fp8_python_refusals():
    x = torch.zeros((4, 300), dtype=torch.bfloat16)
    w = torch.zeros((40, 300), dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros((1, 3), dtype=torch.uint8).view(torch.float8_e8m0fnu)
    for bad in (w.view(torch.uint8), w[:, :299], w[0], w[:0]):
        with pytest.raises(ValueError, match="fp8 weight"):
            cr.fp8_linear(x, bad, s)
    for bad in (s.view(torch.uint8), s[:, :2], s[0]):
        with pytest.raises(ValueError, match="fp8 weight scales"):
            cr.fp8_linear(x, w, bad)
    with pytest.raises(ValueError, match="bias"):
        cr.fp8_linear(x, w, s, torch.zeros(41))
    with pytest.raises(ValueError, match="frozen"):
        cr.fp8_linear(x, w, s, torch.zeros(40, requires_grad=True))
    with pytest.raises(ValueError, match="CUDA"):
        cr.fp8_linear(x, w, s)
    with pytest.raises(ValueError, match="CUDA"):
        cr.quantize_fp8_weight(x)
    with pytest.raises(ValueError, match="unsupported dtype"):
        cr.quantize_fp8_blockwise(x.double())
    with pytest.raises(ValueError, match="positive sizes"):
        cr.Fp8Linear(0, 4)
    layer = cr.Fp8Linear(300, 40).bfloat16()
    assert layer.qweight.dtype == layer.scales.dtype == torch.uint8 and layer.bias.dtype == torch.float32
    with pytest.raises(ValueError, match="expected K=300"):
        layer(x[:, :200])


# --- AdamW and the gradient norm ----------------------------------------------


class _AdamWTensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "scales")] + [("numel", ctypes.c_int64)]


class _AdamWOptions(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("step", "lr", "beta1", "beta2", "eps", "weight_decay")] + [
        ("step_device", ctypes.c_void_p), ("lr_device", ctypes.c_void_p), ("sums", ctypes.c_void_p),
        ("sums_count", ctypes.c_int64), ("max_norm", ctypes.c_double), ("norm", ctypes.c_void_p)]


class _GradTensor(ctypes.Structure):
    _fields_ = [("grad", ctypes.c_void_p), ("numel", ctypes.c_int64)]


def test_adamw_arguments(lib):
    def run(count=1, dtype=0, bits=8, tensor=None, options=None, how=True):
        t = dict(param=4096, grad=4096, exp_avg=4096, exp_avg_sq=4096, scales=4096, numel=0)
        o = dict(step=1.0, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0)
        tensors = (_AdamWTensor * 1)(_AdamWTensor(**{**t, **(tensor or {})}))
        return lib.convrot_adamw(count, tensors, dtype, bits, ctypes.byref(_AdamWOptions(**{**o, **(options or {})})) if how else None,
                                 None)

    assert run() == 0 and run(count=0) == 0  # no values: nothing to do
    assert run(dtype=4) == -1 and run(bits=16) == -1 and "8 or 32" in _err(lib)
    assert run(count=-1) == -1 and run(how=False) == -1
    assert lib.convrot_adamw(1, None, 0, 8, ctypes.byref(_AdamWOptions(step=1.0)), None) == -1
    for bad in (dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(weight_decay=-1.0), dict(step=0.0), dict(lr=-1.0),
                dict(lr=float("nan")), dict(sums=4096), dict(sums=4096, sums_count=4, max_norm=-1.0)):
        assert run(options=bad) == -1
    for bad in (dict(numel=-1), dict(numel=4, param=None), dict(numel=4, grad=4098), dict(numel=4, exp_avg=None),
                dict(numel=4, scales=None), dict(numel=4, scales=4097)):
        assert run(tensor=bad) == -1
    assert run(bits=32, tensor=dict(numel=4, exp_avg_sq=4098)) == -1 and "misaligned" in _err(lib)


def test_norm_arguments(lib):
    one = (_GradTensor * 1)(_GradTensor(4096, 10))
    assert lib.convrot_square_sums(1, one, 3, FAKE, 1, None, None) == -1
    assert lib.convrot_square_sums(1, one, 0, None, 1, None, None) == -1 and lib.convrot_square_sums(1, one, 0, FAKE, 0, None, None) == -1
    assert lib.convrot_square_sums(1, (_GradTensor * 1)(_GradTensor(None, 10)), 0, FAKE, 1, None, None) == -1
    assert lib.convrot_square_sums(1, (_GradTensor * 1)(_GradTensor(4097, 10)), 0, FAKE, 1, None, None) == -1
    assert lib.convrot_square_sums(1, one, 0, None, 9, FAKE, None) == -1 and "at most 8" in _err(lib)
    assert lib.convrot_norm_of_sums(FAKE, 0, FAKE, None) == -1 and lib.convrot_norm_of_sums(None, 1, FAKE, None) == -1
    assert lib.convrot_square_sums_count(0, None) == 1
    assert lib.convrot_square_sums_count(1, (_GradTensor * 1)(_GradTensor(None, 256 * 8 * 3 + 1))) == 4


def test_optimizer_refusals():
    p = [torch.nn.Parameter(torch.zeros(10))]
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0),
                dict(max_norm=-1.0)):
        with pytest.raises(ValueError):
            cr.AdamW(p, **bad)
    with pytest.raises(ValueError, match="CUDA"):
        cr.adamw_step([p[0]], [torch.zeros(10)], [torch.zeros(10)], [torch.zeros(10)], None, 1, lr=1e-3)
    with pytest.raises(ValueError, match="CUDA"):
        cr.grad_norm([torch.zeros(3)])
    with pytest.raises(ValueError, match="at least one"):
        cr.grad_norm([])
    with pytest.raises(TypeError):
        cr.adamw_step(3, [], [], [], None, 1, lr=1e-3)
    assert cr.adamw_step([], [], [], [], None, 1, lr=1e-3) is None
    optimizer = cr.AdamW(p)
    assert optimizer.step() is None and not optimizer.state  # no gradients: nothing happens
