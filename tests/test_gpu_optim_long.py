"""AdamW with 8-bit moments over many steps against averages in 64 bits of the same gradients, for the betas that its
documentation names.

Bounds.  A kept root is rounded to nearest each step, by 2^-4 of it at most, and what a step changes by less than that to
the border is lost; with b2 up to 0.95 a step's change (2.5% down without a gradient, more up) and its block's scale move
a code across borders often enough that no such loss adds up: the median is within one rounding, and nine of ten values
within four.  m changes by more than a rounding in nearly every step: 2^-4 of its norm."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import dev
from tests.ops64 import randn
from tests.test_gpu_optim import _decoded

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("change", [1.0, 0.25, 4.0])
@pytest.mark.parametrize("beta2", [0.9, 0.95])
def test_8_bit_moments_follow_their_averages(beta2, change):
    n, steps = 64 * 256, 400
    strength = torch.exp(randn((n,), torch.float32, 1) * 1.5 - 5)
    turning = torch.rand(n, generator=torch.Generator(device=dev()).manual_seed(2), device=dev()) < 0.25
    p = torch.zeros(n, device=dev())
    m, r = (torch.zeros(n, dtype=torch.uint8, device=dev()).view(E4M3) for _ in range(2))
    scales = torch.zeros((n // 256, 2), device=dev())
    m64, v64 = (torch.zeros(n, dtype=torch.float64, device=dev()) for _ in range(2))
    for step in range(1, steps + 1):
        if step == steps // 2:  # the gradients of a quarter of the values fade or grow
            strength = torch.where(turning, strength * change, strength)
        g = randn((n,), torch.float32, 10 + step) * strength
        cr.adamw_step([p], [g], [m], [r], [scales], step, lr=1e-4, betas=(0.9, beta2), weight_decay=0.0)
        m64.mul_(0.9).add_(g, alpha=0.1)
        v64.mul_(beta2).addcmul_(g.double(), g.double(), value=1 - beta2)
    ratio = _decoded(r, scales, 1) / v64.sqrt()
    for part in (ratio[turning], ratio[~turning]):
        low, mid, high = torch.quantile(part, torch.tensor([0.05, 0.5, 0.95], dtype=torch.float64, device=dev())).tolist()
        assert abs(mid - 1) <= 2.0 ** -4 and low >= 1 - 2.0 ** -2 and high <= 1 + 2.0 ** -2, (low, mid, high)
    assert (_decoded(m, scales, 0) - m64).norm() <= 2.0 ** -4 * m64.norm()
