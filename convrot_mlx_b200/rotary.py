"""Rotary positions with several axes (time, height, width) for the queries and keys of image and video attention,
with their gradients.  No counterpart in the reference."""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .core import _dtype_code, _require_cuda

_Strides = ctypes.c_int64 * 12


@functools.lru_cache(maxsize=64)
def _widths(axes: tuple[int, ...]):
    return (ctypes.c_int32 * len(axes))(*axes)


def _turn(q, k, q_out, k_out, positions, axes, theta, interleaved, inverse) -> None:
    b, hq, t, d = q.shape
    if k is None:
        kp = kop = None
        hk, strides = 0, _Strides(*q.stride()[:3], *q_out.stride()[:3])
    else:
        kp, kop, hk = k.data_ptr(), k_out.data_ptr(), k.shape[1]
        strides = _Strides(*q.stride()[:3], *q_out.stride()[:3], *k.stride()[:3], *k_out.stride()[:3])
    _lib.call("convrot_axial_rotary", q.get_device(), _dtype_code(q.dtype), b, t, d, q.data_ptr(), q_out.data_ptr(), hq,
              kp, kop, hk, strides, positions.data_ptr(), positions.stride(0) if positions.ndim == 3 else 0, len(axes),
              _widths(axes), theta, interleaved, inverse)


def _packed(t):
    return None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _unit(t):
    return t if t is None or t.stride(3) == 1 else t.contiguous()


def _forward(q, k, positions, axes, theta, interleaved):
    q, k = _unit(q), _unit(k)
    q_out, k_out = _packed(q), _packed(k)
    _turn(q, k, q_out, k_out, positions, axes, theta, interleaved, False)
    return q_out, k_out


class _AxialRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, axes, theta, interleaved):
        ctx.save_for_backward(positions)
        # the gradients take the memory order of the inputs, often columns of one projection's output
        ctx.how = (axes, theta, interleaved, q.stride(1) < q.stride(2))
        return _forward(q, k, positions, axes, theta, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        axes, theta, interleaved, heads_inside = ctx.how

        def like(g):
            if g is None or not heads_inside:
                return _packed(g)
            b, h, t, d = g.shape
            return torch.empty((b, t, h, d), dtype=g.dtype, device=g.device).transpose(1, 2)

        dq, dk = _unit(dq), _unit(dk)
        q_out, k_out = like(dq), like(dk)
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
    if positions.dtype is not torch.float32 or not positions.is_contiguous():
        positions = positions.detach().to(torch.float32).contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _AxialRotary.apply(q, k, positions, axes, float(theta), bool(interleaved))
    return _forward(q, k, positions, axes, float(theta), bool(interleaved))
