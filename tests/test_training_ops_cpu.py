"""Host-side checks of the 8-bit and training operators (no GPU needed): refusals before any device work, the shapes
that make no work, and the plain names of the package."""

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


def test_quantizer_arguments(lib):
    ok = lambda *a: lib.convrot_quantize_i8(FAKE, *a, None, FAKE, 16, FAKE, None)  # noqa: E731
    assert ok(9, 2, 16, 16) == -1 and "dtype" in _err(lib)
    assert ok(2, -1, 16, 16) == -1 and ok(2, 2, 0, 16) == -1
    assert ok(2, 2, 16, 15) == -1 and "strides" in _err(lib)
    assert ok(2, 2, 17, 17) == -1
    assert ok(2, 0, 16, 16) == 0
    assert lib.convrot_quantize_i8(None, 2, 2, 16, 16, None, FAKE, 16, FAKE, None) == -1


def test_gemm_arguments(lib):
    def run(m=4, n=8, k=16, sa=16, sw=16, layout=0, dtype=2, act=FAKE, weight=FAKE, out=FAKE):
        return lib.convrot_i8_gemm(act, sa, weight, sw, layout, FAKE, FAKE, None, out, dtype, m, n, k, None)

    assert run(layout=2) == -1 and run(dtype=5) == -1
    assert run(m=-1) == -1 and run(n=0) == -1 and run(k=0) == -1
    assert run(sa=8) == -1 and run(sw=24) == -1 and "multiples of 16" in _err(lib)
    assert run(k=32, sw=32) == -1  # the activation's rows do not cover k
    assert run(layout=1, n=40, sw=32) == -1  # (k, n) rows do not cover n
    assert run(k=131073, sa=131088, sw=131088) == -2 and "overflow" in _err(lib)
    assert run(act=ctypes.c_void_p(4098)) == -1 and "aligned" in _err(lib)
    assert run(act=None) == -1
    assert run(m=0) == 0


def test_linear_arguments(lib):
    def run(dtype=2, m=4, k=16, codes=FAKE, pitch=16, x=FAKE, stride=16):
        return lib.convrot_i8_linear(x, dtype, stride, None, FAKE, 16, 0, FAKE, None, FAKE, dtype, m, 8, k, codes,
                                     pitch, FAKE, None)

    assert run(dtype=3) == -1 and run(pitch=24) == -1 and run(codes=None) == -1
    assert run(x=None) == -1 and run(stride=8) == -1 and run(k=131073) == -2
    assert run(m=0) == 0


def test_rotary_arguments(lib):
    strides = (ctypes.c_int64 * 12)()

    def run(widths=(4, 4), dim=8, theta=10000.0, batch=1, tokens=1, dtype=2, heads=1, positions=FAKE):
        w = (ctypes.c_int32 * max(1, len(widths)))(*widths)
        return lib.convrot_axial_rotary(dtype, batch, tokens, dim, FAKE, FAKE, heads, None, None, 0, strides, positions,
                                        0, len(widths), w, theta, 1, 0, None)

    assert run(dtype=3) == -1
    assert run(widths=()) == -1 and run(widths=(2,) * 9, dim=64) == -1 and "axes" in _err(lib)
    assert run(widths=(4, 3)) == -1 and run(widths=(0, 4)) == -1 and run(widths=(4, 6)) == -1
    assert run(theta=0.0) == -1 and run(theta=float("inf")) == -1 and run(theta=float("nan")) == -1
    assert run(dim=258) == -2 and run(dim=0) == -2
    assert run(batch=-1) == -1 and run(positions=None) == -1
    assert run(batch=0) == 0 and run(tokens=0) == 0 and run(heads=0) == 0


def test_norm_arguments(lib):
    def run(dtype=2, wdtype=2, rows=4, features=8, per=4, stride=8, eps=1e-6, x=FAKE, mean=None, rstd=None):
        return lib.convrot_layer_norm(x, dtype, rows, features, FAKE, FAKE, wdtype, per, stride, 0, eps, FAKE, mean,
                                      rstd, None)

    assert run(dtype=4, wdtype=4) == -1 and run(wdtype=1) == -1 and "weight" in _err(lib)
    assert run(rows=-1) == -1 and run(features=0) == -1
    assert run(per=3) == -1 and run(per=0) == -1
    assert run(per=2, stride=7) == -1 and "stride" in _err(lib)
    assert run(eps=-1.0) == -1 and run(x=None) == -1 and run(mean=FAKE) == -1
    assert run(rows=0) == 0
    assert lib.convrot_layer_norm_workspace(0, 8, 1) == 0
    size = lib.convrot_layer_norm_workspace(1000, 640, 1000)
    assert size >= 2 * 640 * 4

    def back(space=FAKE, size=size, x=FAKE):
        return lib.convrot_layer_norm_backward(x, FAKE, 2, 1000, 640, FAKE, 2, 1000, 640, 0, FAKE, FAKE, FAKE, FAKE,
                                               None, space, size, None)

    assert back(space=None) == -1 and back(size=size - 1) == -1 and back(space=ctypes.c_void_p(4100)) == -1
    assert "workspace" in _err(lib) and back(x=None) == -1


def test_gelu_arguments(lib):
    assert lib.convrot_gelu_saved8(FAKE, 3, 2, 4, FAKE, FAKE, FAKE, None) == -1
    assert lib.convrot_gelu_saved8(FAKE, 2, -2, 4, FAKE, FAKE, FAKE, None) == -1
    assert lib.convrot_gelu_saved8(FAKE, 2, 2, 0, FAKE, FAKE, FAKE, None) == -1
    assert lib.convrot_gelu_saved8(FAKE, 2, 2, 4, FAKE, FAKE, None, None) == -1
    assert lib.convrot_gelu_saved8(FAKE, 2, 0, 4, FAKE, FAKE, FAKE, None) == 0
    assert lib.convrot_gelu_saved8_backward(FAKE, 2, 2, 4, None, FAKE, FAKE, None) == -1
    assert lib.convrot_gelu_saved8_backward(FAKE, 2, 0, 4, FAKE, FAKE, FAKE, None) == 0


def test_python_refusals():
    x, w, s = torch.zeros(4, 64), torch.zeros((8, 64), dtype=torch.int8), torch.ones(8)
    with pytest.raises(ValueError, match="CUDA"):
        cr.int8_linear(x, w, s)
    with pytest.raises(ValueError, match="2D int8"):
        cr.int8_linear(x, w.float(), s)
    with pytest.raises(ValueError, match="activation K=64"):
        cr.int8_linear(x, w[:, :32], s)
    with pytest.raises(ValueError, match="weight scales"):
        cr.int8_linear(x, w, s[:4])
    with pytest.raises(ValueError, match="int8 bias"):
        cr.int8_linear(x, w, s, s[:4])
    with pytest.raises(ValueError, match="2D int8 activation"):
        cr.int8_matmul(x, w, s[:4], s, output_dtype=torch.float32)
    with pytest.raises(ValueError, match="activation scales"):
        cr.int8_matmul(x.to(torch.int8), w, s, s, output_dtype=torch.float32)
    with pytest.raises(ValueError, match="unsupported dtype"):
        cr.int8_matmul(x.to(torch.int8), w, s[:4], s, output_dtype=torch.float64)
    with pytest.raises(ValueError, match="2D input"):
        cr.quantize_signed_int8_rowwise(torch.zeros(2, 3, 4))
    with pytest.raises(ValueError, match="weight must be 2D"):
        cr.quantize_int8_weight(torch.zeros(3))
    with pytest.raises(ValueError, match="positive sizes"):
        cr.Int8Linear(0, 4)
    layer = cr.Int8Linear(100, 7)
    assert tuple(layer.qweight.shape) == (7, 112) and set(dict(layer.named_buffers())) == {"qweight", "scales", "bias"}
    with pytest.raises(ValueError, match="expected K=100"):
        layer(torch.zeros(2, 99))
    assert cr.Int8Linear(16, 4, bias=False).bias is None
    q, pos = torch.zeros((1, 2, 4, 8)), torch.zeros((4, 2))
    with pytest.raises(ValueError, match="CUDA"):
        cr.axial_rotary(q, None, pos, (4, 4))
    with pytest.raises(ValueError, match="axis widths"):
        cr.axial_rotary(q, None, pos, (4, 6))
    with pytest.raises(ValueError, match="CUDA"):
        cr.layer_norm(x)
    with pytest.raises(ValueError, match="weight must have shape"):
        cr.layer_norm(x, s)
    with pytest.raises(ValueError, match="modulation vector"):
        cr.modulated_layer_norm(x.view(2, 2, 64), x[:3], x[:2])
    with pytest.raises(ValueError, match="CUDA"):
        cr.gelu_tanh_saved8(x)
