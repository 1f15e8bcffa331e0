"""The input gradient of an 8-bit linear with more channels than one int32 dot can sum (131072), against 64 bits.

Bound: each range's dot is exact; its conversion and scale are two float32 roundings, the join one for each range and
one to the output: 4 U of the ranges' magnitudes.  Codes as in test_gpu_int8.py."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import assert_no_device_error
from tests.ops64 import DTYPES, U, assert_within, codes64, randn

pytestmark = pytest.mark.gpu
RANGE = 131072


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(2, 48, RANGE + 1), (1, 17, 400001), (200, 40, 2 * RANGE + 16), (0, 32, RANGE + 3)])
def test_input_gradient_over_many_channels(dtype, m, k, n):
    qweight, wscales = cr.quantize_int8_weight(randn((n, k), torch.float32, 11, 0.05))
    x = randn((m, 1, k), dtype, 12).requires_grad_()
    y = cr.int8_linear(x, qweight, wscales)
    assert torch.equal(y.detach()[:, :, -40:], cr.int8_linear(x.detach(), qweight[-40:], wscales[-40:]))
    dy = randn((m, 1, n), dtype, 13, 0.1)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert dx.shape == x.shape and dx.dtype == dtype
    if m == 0:
        return
    q, c, s = codes64((dy.float() * wscales)[:, 0].double())
    near = ((q - q.floor() - 0.5).abs() < 2e-5).double()
    w = qweight.double()
    parts = [c[:, at:at + RANGE] @ w[at:at + RANGE] * s for at in range(0, n, RANGE)]
    slack = 4 * U * sum(p.abs() for p in parts) + near @ w.abs() * s
    assert_within(dx[:, 0], sum(parts), slack, f"{m} {k} {n}")
    assert_no_device_error()
