"""Activations of a training step whose saved input is held in 8 bits.  No counterpart in the reference."""

from __future__ import annotations

import torch

from . import _native


def gelu_tanh_saved8(x: torch.Tensor) -> torch.Tensor:
    """Tanh GELU whose backward pass reads its input from 8 bits.

    The output is that of the input as given; for the backward pass only int8
    codes of x are kept, with one float32 scale for each 128 features of a
    row: about half of a 16-bit x, and none of x itself.  The gradient is the
    formula's at the restored input, at most half a code step (1/254 of its
    group's largest magnitude) away."""

    return _native.ops().gelu_tanh_saved8(x)
