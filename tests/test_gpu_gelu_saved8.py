"""The tanh GELU whose saved input is held in 8 bits (convrot_gelu_saved8, gelu_tanh_saved8) against 64-bit arithmetic.

Bounds.  y = x s(x): the exponent is a float32 expression of magnitude at most e = 2 |u| with 4 roundings, and the
exponential and division intrinsics are within 2^-21 plus 2^-22 e, so s is relatively off by at most 12 U (1 + e),
U = 2^-24 (where s itself is below the float32 range the product is too).  The slope adds a handful of roundings:
32 U (1 + e) of the sum of its terms' magnitudes."""

from __future__ import annotations

import math

import pytest
import torch

import convrot_mlx_b200 as cr
from convrot_mlx_b200 import _lib
from tests.gpu_util import assert_no_device_error, dev
from tests.ops64 import DTYPES, U, assert_within, codes64, randn

pytestmark = pytest.mark.gpu
C, A, GROUP = math.sqrt(2 / math.pi), 0.044715, 128


def _y64(x):
    x = x.double()
    e = 2 * C * (x + A * x ** 3)
    y = x * torch.sigmoid(e)
    return y, 12 * U * (1 + e.abs()) * y.abs() + 1e-38


def _slope64(r):
    e = 2 * C * (r + A * r ** 3)
    s, t = torch.sigmoid(e), torch.sigmoid(-e)
    second = r * s * t * 2 * C * (1 + 3 * A * r * r)
    # 1 - s is formed from the rounded s: an absolute error of one more s-error
    err = 12 * U * (1 + e.abs()) * s
    return s + second, 32 * U * (1 + e.abs()) * (s + second.abs()) + err * (r * 2 * C * (1 + 3 * A * r * r)).abs() + 1e-38


def _restored64(x):
    """The restored input in 64 bits, and where a float32 input's code may go either way, by one step."""

    f = x.shape[-1]
    groups = torch.nn.functional.pad(x.double(), (0, -f % GROUP)).unflatten(-1, (-1, GROUP))
    q, c, s = codes64(groups)
    unsure = ((q - q.floor() - 0.5).abs() < 2e-5) & (x.dtype == torch.float32)
    step = torch.where(unsure, s.expand_as(q), torch.zeros_like(q))
    return (c * s).flatten(-2)[..., :f], step.flatten(-2)[..., :f]


def _check(x, y, dy, dx):
    assert_within(y, *_y64(x), "y")
    r, step = _restored64(x)
    slope, err = _slope64(r)
    # restoring rounds twice (the scale and the product): 2.1 U |r| against a slope of slope at most 1.13
    err = err + 1.13 * (2.1 * U * r.abs() + 1.1 * step)
    assert_within(dx, dy.double() * slope, dy.double().abs() * (err + 2 * U * slope.abs()), "dx")


SHAPES = [(1, 1), (3, 7), (2, 127), (2, 128), (5, 129), (4, 256), (1, 12288), (33, 4100), (500, 96), (17, 1000), (300, 513),
          (9, 16384), (64, 2056), (5, 258), (40, 1030), (700, 384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", SHAPES)
def test_forward_and_gradient(dtype, rows, features):
    x = randn((rows, features), dtype, rows + features, 2.0).requires_grad_()
    dy = randn((rows, features), dtype, 2)
    y = cr.gelu_tanh_saved8(x)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert y.dtype == dx.dtype == dtype
    _check(x.detach(), y.detach(), dy, dx)
    assert torch.equal(y.detach(), cr.gelu_tanh_saved8(x.detach()))  # without a gradient: the same values
    assert_no_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
def test_outliers_zero_groups_and_saturated_values(dtype):
    x = randn((6, 400), dtype, 3)
    x[0, :128] = 0
    x[1] = 0
    x[2, ::7] *= 30
    x[3] = 60.0
    x[4] = -60.0
    x[5, 200] = 6.0e4
    x.requires_grad_()
    dy = randn(x.shape, dtype, 4)
    y = cr.gelu_tanh_saved8(x)
    _check(x.detach(), y.detach(), dy, torch.autograd.grad(y, x, dy)[0])


def test_values_near_the_end_of_the_type():
    big = 1.0e38
    x = torch.tensor([[big, -big, 1.0, 0.0]], dtype=torch.bfloat16, device=dev(), requires_grad=True)
    y = cr.gelu_tanh_saved8(x)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(x))
    assert y[0, 0] == x[0, 0] and y[0, 1] == 0
    assert dx[0].tolist() == [1.0, 0.0, 0.5, 0.5]  # beside 1e38 the others are restored as 0


def test_groups_that_are_not_finite():
    x = randn((2, 384), torch.bfloat16, 5)
    x[0, 130], x[1, 300] = float("nan"), float("inf")
    x.requires_grad_()
    y = cr.gelu_tanh_saved8(x)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(x))
    assert torch.isnan(y[0, 130]) and y[1, 300] == float("inf")
    bad = torch.zeros((2, 384), dtype=torch.bool, device=dev())
    bad[0, 128:256], bad[1, 256:] = True, True
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()


def test_gradient_against_differences():
    # inputs that their codes give back exactly (127 steps of a power of two), so that the slope is that of the output
    x = torch.arange(-127, 129, device=dev()).clamp(max=127).float().view(2, 128) / 32
    x[0, 1], x[1, 0] = 127 / 32, -127 / 32
    x.requires_grad_()
    (dx,) = torch.autograd.grad(cr.gelu_tanh_saved8(x), x, torch.ones_like(x))
    e = 1e-2
    d = (cr.gelu_tanh_saved8(x.detach() + e).double() - cr.gelu_tanh_saved8(x.detach() - e).double()) / (2 * e)
    # third derivative at most 2.5, e^2 / 6 of it; the float32 rounding of values up to 4 over the step
    assert (dx.double() - d).abs().max() <= 2.5 * e * e / 6 + 16 * U * 4 / e


def test_memory_that_is_kept():
    x = randn((1024, 4096), torch.bfloat16, 6).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = cr.gelu_tanh_saved8(x)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert kept <= x.numel() * (1 + 4 / 128) + 4096


def test_shapes_strides_empty_and_expanded():
    base = randn((4, 6, 300), torch.bfloat16, 7)
    for v in (base[..., 1:], base[:, ::2], base.transpose(0, 1), base[0, 0]):
        v = v.detach().requires_grad_()
        w = v.detach().contiguous().clone().requires_grad_()
        a, c = cr.gelu_tanh_saved8(v), cr.gelu_tanh_saved8(w)
        assert a.shape == v.shape and torch.equal(a, c)
        assert torch.equal(torch.autograd.grad(a.sum(), v)[0], torch.autograd.grad(c, w, torch.ones_like(c))[0])
    e = torch.empty((0, 5), device=dev(), requires_grad=True)
    assert torch.autograd.grad(cr.gelu_tanh_saved8(e).sum(), e)[0].shape == (0, 5)


def test_unaligned_rows_through_the_c_entry():
    # addresses and widths for which no wide access is aligned
    rows, f = 5, 260
    x = randn((rows * f + 1,), torch.bfloat16, 8)[1:].view(rows, f)
    y = torch.empty((rows * f + 1,), dtype=torch.bfloat16, device=dev())[1:].view(rows, f)
    codes = torch.empty((rows * f + 3,), dtype=torch.int8, device=dev())[3:].view(rows, f)
    scales = torch.empty((rows, 3), device=dev())
    _lib.call("convrot_gelu_saved8", 0, x.data_ptr(), _lib.BF16, rows, f, y.data_ptr(), codes.data_ptr(),
              scales.data_ptr())
    dx = torch.empty_like(x)
    _lib.call("convrot_gelu_saved8_backward", 0, x.data_ptr(), _lib.BF16, rows, f, codes.data_ptr(), scales.data_ptr(),
              dx.data_ptr())
    _check(x, y, x, dx)
    groups = torch.nn.functional.pad(x.double(), (0, -f % GROUP)).unflatten(-1, (-1, GROUP))
    assert torch.equal(codes.double(), codes64(groups)[1].flatten(-2)[:, :f])


def test_offsets_past_32_bits():
    rows, f = 2 ** 15 + 1, 2 ** 16 + 8
    x = randn((rows, f), torch.bfloat16, 9).requires_grad_()
    y = cr.gelu_tanh_saved8(x)
    (dx,) = torch.autograd.grad(y, x, y.detach())
    for part in (slice(0, 2), slice(rows - 2, rows)):
        _check(x.detach()[part], y.detach()[part], y.detach()[part], dx[part])


def test_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        cr.gelu_tanh_saved8(torch.zeros(2, 3))
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        cr.gelu_tanh_saved8(torch.zeros((2, 3), dtype=torch.float64, device=dev()))
    with pytest.raises(ValueError, match="features"):
        cr.gelu_tanh_saved8(torch.zeros((2, 0), device=dev()))
    p = _lib.ptr(torch.zeros((2, 4), device=dev()))
    lib = _lib.load()
    assert lib.convrot_gelu_saved8(p, 7, 2, 4, p, p, p, None) == -1
    assert lib.convrot_gelu_saved8(p, 0, 2, 4, p, p, None, None) == -1
    assert lib.convrot_gelu_saved8_backward(p, 0, 2, 4, None, p, p, None) == -1


def test_a_gradient_that_would_be_differentiated_again_is_refused():
    x = randn((4, 8), torch.float32, 1).requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(cr.gelu_tanh_saved8(x).sum(), x, create_graph=True)
    w = torch.ones(8, device=dev())
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(cr.layer_norm(x, w).sum(), x, create_graph=True)
