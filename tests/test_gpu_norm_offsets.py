"""Layer norm of constant and nearly constant rows far from zero, against 64-bit arithmetic.

Bounds.  E = (F / 32 + 24) U is the relative error of a row's sum (test_gpu_norm.py), X = max|x|, dev = max|x - mean|.
The first mean is off by delta <= E X, so the centred values are at most D = dev + E X (each rounded once); where the
mean is beyond twice the deviation their own mean, which is off by at most E D, corrects it, elsewhere delta stays.
Hence
  h = (x - mean) r by dh = r ((E + 4 U) D + 2 U E X) + |h| rel, D being at least X in rows near zero, with rel the
  relative error of r: the sum of squares is off by (E + 4 U) (var + delta^2) and the square of the correction by
  2 E X E D + 2 U (E X)^2 (near zero, by all of delta^2); half of that over var + eps, and 6 U.
The mean that the backward pass reads is rounded to float32 once, U X: its h is off by r U X more, but of a constant row
it is the row's value itself (E D is less than half its last place), so its h is 0."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import assert_no_device_error, dev
from tests.ops64 import U, assert_within, randn

pytestmark = pytest.mark.gpu
EPS = 1e-6
WIDTHS = [64, 700, 1153, 1664, 3000, 5001, 9000, 16384, 20001, 40000, 110001]


def _norm64(x):
    x = x.double()
    E = (x.shape[-1] / 32 + 24) * U
    X = x.abs().amax(-1, keepdim=True)
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    var = c.square().mean(-1, keepdim=True)
    r = (var + EPS).rsqrt()
    h = c * r
    D, delta = c.abs().amax(-1, keepdim=True) + E * X, E * X
    near = mean.abs() * r <= 2.01
    D = torch.where(near, torch.maximum(D, X), D)
    square = torch.where(near, delta ** 2, 2 * delta * E * D + 2 * U * delta ** 2)
    rel = 0.6 * ((E + 4 * U) * (var + delta ** 2) + square) / (var + EPS) + 6 * U
    dh = r * ((E + 4 * U) * D + 2 * U * delta) + h.abs() * rel
    return h, dh, dh + r * U * X, r, rel, E


def _check(x, w, b, dy, constant):
    x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = cr.layer_norm(x, w, b, EPS)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x, w, b = x.detach(), w.detach().double(), b.detach().double()
    h, dh, back, r, rel, E = _norm64(x)
    assert_within(y.detach(), h * w + b, w.abs() * dh + 2 * U * ((h * w).abs() + b.abs()), "y")
    g = dy.double() * w
    m, mh = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    if constant:
        assert dw.eq(0).all()
        back = torch.zeros_like(back)
    G, GH = g.abs().mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    off = (g.abs() * back).mean(-1, keepdim=True)
    parts = 3 * U * g.abs() + (E + 2 * U) * G + h.abs() * ((E + 4 * U) * GH + off) + back * (mh.abs() + off)
    assert_within(dx, r * (g - m - h * mh), r * parts + (rel + 8 * U) * r * (g.abs() + m.abs() + (h * mh).abs()), "dx")
    d, n = dy.double(), x.shape[0]
    assert_within(dw, (d * h).sum(0), (n + 600) * U * (d * h).abs().sum(0) + (d.abs() * back).sum(0), "dw")
    assert_within(db, d.sum(0), (n + 600) * U * d.abs().sum(0), "db")
    assert_no_device_error()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("features", WIDTHS)
def test_constant_rows(dtype, features):
    values = torch.tensor([1.0, 30000.0, -1000.1, 0.0, 12345.678, -3.3], device=dev()).to(dtype)
    x = values[:, None].repeat(1, features)
    w, b = randn((features,), torch.float32, 1), randn((features,), torch.float32, 2)
    dy = randn(x.shape, dtype, 3)
    _check(x, w, b, dy, True)


@pytest.mark.parametrize("spread", [1.0, 0.05])
@pytest.mark.parametrize("features", WIDTHS)
def test_nearly_constant_rows(features, spread):
    x = torch.tensor([1.0, 30000.0, -1000.1, 0.0, 12345.678], device=dev())[:, None] + randn((5, features), torch.float32, 4, spread)
    w, b = randn((features,), torch.float32, 1), randn((features,), torch.float32, 2)
    _check(x, w, b, randn(x.shape, torch.float32, 3), False)


def test_rows_of_sixteen_bits_far_from_zero():
    x = (1000 + 20 * randn((64, 1664), torch.float32, 5)).to(torch.bfloat16)
    w, b = randn((1664,), torch.bfloat16, 1), randn((1664,), torch.bfloat16, 2)
    _check(x, w, b, randn(x.shape, torch.bfloat16, 3), False)
