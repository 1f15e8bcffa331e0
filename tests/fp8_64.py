"""The 8-bit floating-point linear in 64 bits: what its tests compare with."""

from __future__ import annotations

import torch

SPAN = 128


def e4m3(v):
    """v (64 bits) to the nearest e4m3 value, ties to even: steps of 2^(e - 3) in [2^e, 2^(e + 1)), of 2^-9 below 2^-6."""

    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exponent(top):
    """The least e >= -127 with top <= 448 * 2^e; -127 for 0."""

    fraction, e = torch.frexp(top)
    e = e - 9 + (fraction > 0.875).int()
    return torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)


def rows64(x):
    """(codes, exponents) of the blocks of 128 values of each row of x."""

    x64 = x.double()
    k = x.shape[1]
    blocks = torch.nn.functional.pad(x64, (0, -k % SPAN)).unflatten(1, (-1, SPAN))
    e = exponent(blocks.abs().amax(-1))
    return e4m3(blocks * torch.exp2(-e.double())[..., None]).flatten(1)[:, :k], e


def blocks64(w):
    """(codes, exponents) of the 128 x 128 blocks of w."""

    w64 = w.double()
    n, k = w.shape
    blocks = torch.nn.functional.pad(w64, (0, -k % SPAN, 0, -n % SPAN)).unflatten(1, (-1, SPAN)).unflatten(0, (-1, SPAN))
    e = exponent(blocks.abs().amax((1, 3)))
    return e4m3(blocks * torch.exp2(-e.double())[:, None, :, None]).flatten(0, 1).flatten(1)[:n, :k], e


def values_of_rows(codes, scales):
    return codes.double() * scales.float().double().repeat_interleave(SPAN, 1)[:, :codes.shape[1]]


def values_of_blocks(codes, scales):
    n, k = codes.shape
    return codes.double() * scales.float().double().repeat_interleave(SPAN, 0)[:n].repeat_interleave(SPAN, 1)[:, :k]


def product64(a, w, bias=None):
    """(a @ w.T + bias, bound of the 32-bit sums).  A product of two codes has 8 significant bits and is exact; the tensor
    core adds 32 of them to its 32-bit sum in one step, which drops bits below the sum's last one or two: 2^-22 of the
    magnitudes added so far a step, over k / 32 steps, and as much again for the steps' own additions and a split K."""

    core, size = a @ w.T, a.abs() @ w.abs().T
    steps = -(-a.shape[1] // 32) + 32
    y = core if bias is None else core + bias.double()
    return y, steps * 2.0 ** -22 * size + 2.0 ** -24 * y.abs()
