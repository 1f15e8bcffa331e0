"""Rotary positions with several axes (time, height, width) for the queries and keys of image and video attention,
with their gradients.  No counterpart in the reference."""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .core import _dtype_code, _require_cuda

MAX_HEAD_DIM = 256


def _strides(t: torch.Tensor | None):
    return None if t is None else (ctypes.c_int64 * 3)(*t.stride()[:3])


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 else t.contiguous()


def _turn(q, k, q_out, k_out, positions, axes, theta, interleaved, inverse) -> None:
    b, hq, t, d = q.shape
    per_sample = positions.stride(0) if positions.ndim == 3 else 0
    _lib.call("convrot_axial_rotary", q, _dtype_code(q.dtype), b, t, d, _lib.ptr(q), hq, _strides(q), _lib.ptr(q_out),
              _strides(q_out), _lib.ptr(k), 0 if k is None else k.shape[1], _strides(k), _lib.ptr(k_out),
              _strides(k_out), _lib.ptr(positions), per_sample, len(axes), (ctypes.c_int32 * len(axes))(*axes), theta,
              int(interleaved), int(inverse))


def _forward(q, k, positions, axes, theta, interleaved):
    q = _unit(q)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = None
    if k is not None:
        k = _unit(k)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    _turn(q, k, q_out, k_out, positions, axes, theta, interleaved, False)
    return q_out, k_out


class _AxialRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, axes, theta, interleaved):
        ctx.save_for_backward(positions)
        ctx.how = (axes, theta, interleaved)
        # the gradients take the memory order of the inputs, often columns of one projection's output
        ctx.like = q.stride(1) < q.stride(2)
        return _forward(q, k, positions, axes, theta, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        axes, theta, interleaved = ctx.how

        def like(g):
            b, h, t, d = g.shape
            if ctx.like:
                return torch.empty((b, t, h, d), dtype=g.dtype, device=g.device).transpose(1, 2)
            return torch.empty(g.shape, dtype=g.dtype, device=g.device)

        dq = _unit(dq)
        q_out, k_out = like(dq), None
        if dk is not None:
            dk = _unit(dk)
            k_out = like(dk)
        _turn(dq, dk, q_out, k_out, positions, axes, theta, interleaved, True)
        return q_out, k_out, None, None, None, None


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

    axes = tuple(int(w) for w in axes)
    for t, name in ((q, "queries"), (k, "keys")):
        if t is not None and t.ndim != 4:
            raise ValueError(f"rotary {name} must be (batch, heads, tokens, dim), got {tuple(t.shape)}")
    if k is not None and (k.dtype != q.dtype or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]):
        raise ValueError(f"queries {tuple(q.shape)} {q.dtype} and keys {tuple(k.shape)} {k.dtype} do not match")
    b, _, t, d = q.shape
    if not axes or any(w <= 0 or w % 2 for w in axes) or sum(axes) > d:
        raise ValueError(f"axis widths must be positive, even and sum to at most the head dimension {d}, got {axes}")
    if positions.shape not in ((t, len(axes)), (b, t, len(axes))):
        raise ValueError(f"positions must be ({t}, {len(axes)}) or ({b}, {t}, {len(axes)}), got "
                         f"{tuple(positions.shape)}")
    _dtype_code(q.dtype)
    _require_cuda(q, k, positions)
    positions = positions.detach().to(torch.float32).contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _AxialRotary.apply(q, k, positions, axes, float(theta), bool(interleaved))
    return _forward(q, k, positions, axes, float(theta), bool(interleaved))
