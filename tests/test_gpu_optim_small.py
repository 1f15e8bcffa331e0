"""AdamW where the squares of the gradients are below float32's normal range, with eps 0 and above.

Bounds.  v: 5 U of it as for larger values, and three products that are rounded to multiples of 2^-149: within 2^-148.  Its
root moves by at most the error of v over the root; the update by at most the error of v over v, d, beside the 16 U of
the operations: a quotient whose denominator is off by d is off by d / (1 - d)."""

from __future__ import annotations

import math

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import dev
from tests.ops64 import TINY, U, assert_within, randn
from tests.test_gpu_optim import _as_8_bits, _blocks, _check_codes, _decoded

pytestmark = pytest.mark.gpu

BETAS = (0.9, 0.9)


def _gradients(size, n, seed):
    """Between one and three times ``size``, of either sign."""

    g = randn((n,), torch.float32, seed)
    return torch.sign(g) * (1 + g.abs().clamp(max=2)) * size


@pytest.mark.parametrize("eps", [0.0, 1e-8])
@pytest.mark.parametrize("size", [1e-18, 1e-19, 1e-20, 3e-21])
@pytest.mark.parametrize("step", [1, 40])
@pytest.mark.parametrize("bits", [32, 8])
def test_squares_below_the_normal_range(bits, step, size, eps):
    n = 1000
    g = _gradients(size, n, 1)
    p = randn((n,), torch.float32, 2) * (0.1 if eps == 0 else 1e-12 * size / 1e-18)
    m = _gradients(size, n, 3) * (step > 1)
    v = (_gradients(size, n, 4).double() ** 2).float() * (step > 1)
    scales = None
    if bits == 8:
        m, v, scales = _as_8_bits(m, v)
        m64, v64 = _decoded(m, scales, 0), _decoded(v, scales, 1) ** 2
    else:
        m64, v64 = m.double(), v.double()
    p64, g64 = p.double(), g.double()
    cr.adamw_step([p], [g], [m], [v], None if bits == 32 else [scales], step, lr=0.01, betas=BETAS, eps=eps, weight_decay=0.0)
    b1, b2 = BETAS
    m_slack = 4 * U * (b1 * m64.abs() + (1 - b1) * g64.abs())
    m64, v64 = b1 * m64 + (1 - b1) * g64, b2 * v64 + (1 - b2) * g64 * g64
    v_slack = 5 * U * v64 + 2.0 ** -148 + (4 * U * v64 if bits == 8 else 0.0)
    if bits == 32:
        assert_within(m, m64, m_slack)
        assert_within(v, v64, v_slack)
    else:
        root = v64.sqrt()
        _check_codes(_blocks(m), scales[:, 0], _blocks(m64), _blocks(m_slack) + 2 * U * _blocks(m64).abs())
        _check_codes(_blocks(v), scales[:, 1], _blocks(root), _blocks(5 * U * root + v_slack / root), root=True)
    size64 = 0.01 / (1 - b1 ** step)
    den = v64.sqrt() / math.sqrt(1 - b2 ** step) + eps
    update = size64 * m64 / den
    d = v_slack / v64 / (1 - v_slack / v64)
    slack = 4 * U * p64.abs() + update.abs() * (16 * U + d) + size64 / den * m_slack * (1 + d) + TINY[torch.float32]
    assert_within(p, p64 - update, slack)


def test_zeros_among_small_and_large_squares():
    # a thread's eight values of all sizes at once: each as if it were alone
    n = 512
    size = torch.tensor([0.0, 1e-22, 1e-20, 1e-19, 1e-10, 1.0, 1e10, 1e18], device=dev()).repeat(n // 8)
    for order in range(8):
        g = size.roll(order) * torch.sign(randn((n,), torch.float32, 7 + order))
        p, m, v = (torch.zeros(n, device=dev()) for _ in range(3))
        cr.adamw_step([p], [g], [m], [v], None, 1, lr=1.0, betas=(0.9, 0.5), eps=0.0, weight_decay=0.0)
        assert torch.isnan(p[g == 0]).all()  # 0 / 0
        for value in size.unique()[2:]:
            of = g.abs() == value  # the first update is the gradient's sign, but for v's rounding
            v64 = 0.5 * g[of].double() ** 2
            d = (2.0 ** -148 + 5 * U * v64) / v64
            assert ((p[of].double() + torch.sign(g[of]).double()).abs() <= 20 * U + d / (1 - d)).all(), value
