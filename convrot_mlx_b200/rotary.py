"""Rotary positions with several axes (time, height, width) for the queries and keys of image and video attention,
with their gradients.  No counterpart in the reference."""

from __future__ import annotations

import torch

from . import _native


def axial_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, axes, *, theta: float = 10000.0,
                 interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Queries and keys turned by their tokens' positions along several axes.

    q: (batch, heads, tokens, dim) and k: (batch, key heads, tokens, dim) or
    None, of any strides (views of a fused projection's output are read in
    place); positions: (tokens, len(axes)) or (batch, tokens, len(axes)),
    taken as float32.  ``axes`` gives the width of each axis: the first
    sum(axes) values of a head form pairs, adjacent ones with ``interleaved``,
    else sum(axes) / 2 apart; axis a owns axes[a] / 2 consecutive pairs, and
    its pair j turns by positions[..., a] * theta ** (-2 j / axes[a]).  The
    rest of a head is copied.  Returns new packed (batch, heads, tokens, dim)
    tensors; differentiable in q and k."""

    return _native.ops().axial_rotary(q, k, positions, axes, theta, interleaved)
