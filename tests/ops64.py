"""What the tests of the 8-bit and training operators share: seeded inputs and rounding bounds.

``HALF[dtype]`` is the largest relative error of one rounding to that type, ``TINY[dtype]`` half its smallest
subnormal; ``U`` is the float32 one, in which the kernels calculate."""

from __future__ import annotations

import torch

from tests.gpu_util import dev

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=dev()).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev()) * scale).to(dtype)


def assert_within(got, want64, slack64, what=""):
    """|got - want| <= one rounding of got's type + slack (the float32 arithmetic's share), element by element."""

    bound = HALF[got.dtype] * want64.abs() + TINY[got.dtype] + slack64 * (1 + HALF[got.dtype])
    off = (got.double() - want64).abs()
    assert torch.isfinite(got.double()).all(), what
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: off by {off.max().item():.3g}, {worst:.3g} over its bound"


def codes64(x64):
    """The 8-bit quantizer in 64 bits: the exact quotients 127 x / top, their rounding, and the scales."""

    top = x64.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, 127 * x64 / top, torch.zeros_like(x64))
    return q, q.round(), top / 127
