"""Rotary positions with several axes (convrot_axial_rotary, axial_rotary) against 64-bit arithmetic.

Bound.  The angle is formed in 64 bits and handed over as a float32 fraction of a turn (2^-24 of half a turn: an angle
error of at most pi 2^-24), sine and cosine are within 2 ulps (2^-22), and two products and a sum of float32 round
three times: less than 8 * 2^-24 (|x0| + |x1|) in all, plus the rounding of the output."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import assert_no_device_error, dev
from tests.ops64 import DTYPES, U, assert_within, randn

pytestmark = pytest.mark.gpu


def _rotate64(x, positions, axes, theta, interleaved, sign=1.0):
    x = x.double()
    pos = positions.double()
    pos = pos if pos.ndim == 3 else pos[None]
    ang = torch.cat([pos[..., a, None] * theta ** (-2.0 * torch.arange(w // 2, device=dev()).double() / w)
                     for a, w in enumerate(axes)], -1)[:, None] * sign
    n = ang.shape[-1]
    x0, x1 = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    y0, y1 = x0 * ang.cos() - x1 * ang.sin(), x0 * ang.sin() + x1 * ang.cos()
    y, slack = x.clone(), torch.zeros_like(x)
    s = 8 * U * (x0.abs() + x1.abs())
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2], slack[..., 0:2 * n:2], slack[..., 1:2 * n:2] = y0, y1, s, s
    else:
        y[..., :n], y[..., n:2 * n], slack[..., :n], slack[..., n:2 * n] = y0, y1, s, s
    return y, slack


def _positions(tokens, axes, seed, top=100):
    g = torch.Generator(device=dev()).manual_seed(seed)
    return torch.randint(0, top, (tokens, len(axes)), generator=g, device=dev()).float()


CASES = [  # batch, heads, key heads, tokens, dim, axes
    (1, 1, 1, 1, 2, (2,)),
    (2, 3, 1, 5, 8, (4, 2)),
    (1, 24, 24, 40, 128, (16, 56, 56)),
    (2, 6, 2, 77, 128, (32, 40, 40)),
    (3, 4, 4, 33, 64, (20, 20)),
    (1, 5, 1, 130, 256, (42, 84, 84)),
    (1, 2, 2, 9, 30, (6, 10, 6)),
    (2, 3, 3, 11, 37, (6, 10, 14)),
    (1, 8, 2, 300, 96, (16, 32, 32)),
    (1, 1, 1, 3000, 72, (24, 24, 24)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,h,kv,t,d,axes", CASES)
def test_forward_and_gradient(dtype, interleaved, b, h, kv, t, d, axes):
    q, k = randn((b, h, t, d), dtype, 1).requires_grad_(), randn((b, kv, t, d), dtype, 2).requires_grad_()
    pos = _positions(t, axes, 3)
    yq, yk = cr.axial_rotary(q, k, pos, axes, theta=10000.0, interleaved=interleaved)
    assert yq.shape == q.shape and yk.shape == k.shape and yq.is_contiguous() and yk.is_contiguous()
    for x, y in ((q, yq), (k, yk)):
        assert_within(y.detach(), *_rotate64(x.detach(), pos, axes, 10000.0, interleaved))
    dq, dk = randn(q.shape, dtype, 4), randn(k.shape, dtype, 5)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    for x, y in ((dq, gq), (dk, gk)):
        assert_within(y, *_rotate64(x, pos, axes, 10000.0, interleaved, -1.0))
    assert_no_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,axes", [(128, (16, 56, 56)), (64, (8, 24, 24)), (40, (8, 12, 12))])
def test_views_of_a_projection(dtype, interleaved, d, axes):
    b, t, h, kv = 2, 50, 6, 2
    pos = _positions(t, axes, 6)
    for pad in (0, 1, 8):  # columns of a wider row; with 1 nothing is aligned
        qkv = randn((b, t, (h + 2 * kv) * d + pad), dtype, 7)
        heads = qkv[..., pad:].unflatten(-1, (-1, d))
        q, k = heads[:, :, :h].transpose(1, 2), heads[:, :, h:h + kv].transpose(1, 2)
        q.requires_grad_(), k.requires_grad_()
        yq, yk = cr.axial_rotary(q, k, pos, axes, theta=256.0, interleaved=interleaved)
        assert_within(yq.detach(), *_rotate64(q.detach(), pos, axes, 256.0, interleaved))
        assert_within(yk.detach(), *_rotate64(k.detach(), pos, axes, 256.0, interleaved))
        dq = randn((b, t, h, d), dtype, 8).transpose(1, 2)  # a gradient in the other memory order
        gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, torch.ones_like(yk[:, :1]).expand_as(yk)))
        assert_within(gq, *_rotate64(dq, pos, axes, 256.0, interleaved, -1.0))
        assert_within(gk, *_rotate64(torch.ones_like(yk).detach(), pos, axes, 256.0, interleaved, -1.0))
    assert_no_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,axes", [(8, (2,)), (8, (6,)), (16, (14,)), (64, (10, 20, 20)), (64, (2, 4)), (88, (30, 30, 26)),
                                    (96, (42, 42)), (128, (20, 42, 42)), (128, (126,)), (132, (44, 42, 42)),
                                    (136, (40, 42, 42)), (248, (2,)), (256, (42, 84, 84)), (256, (86, 84, 86))])
@pytest.mark.parametrize("t,h,kv", [(1, 1, 1), (3, 40, 8), (37, 5, 2), (260, 13, 25)])
def test_halves_that_begin_anywhere(dtype, d, axes, t, h, kv):
    b = 2
    q, k = randn((b, h, t, d), dtype, 41).requires_grad_(), randn((b, kv, t, d), dtype, 42).requires_grad_()
    pos = _positions(t, axes, 43)
    yq, yk = cr.axial_rotary(q, k, pos, axes, interleaved=False)
    for x, y in ((q, yq), (k, yk)):
        assert_within(y.detach(), *_rotate64(x.detach(), pos, axes, 10000.0, False))
    dq, dk = randn(q.shape, dtype, 44), randn(k.shape, dtype, 45)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    for x, y in ((dq, gq), (dk, gk)):
        assert_within(y, *_rotate64(x, pos, axes, 10000.0, False, -1.0))
    assert_no_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,axes", [(64, (10, 20, 20)), (128, (32, 40, 40)), (37, (6, 10, 14))])
def test_values_past_the_pairs_are_copied(dtype, interleaved, d, axes):
    turned = sum(axes)
    q = randn((1, 3, 20, d), dtype, 51)
    q[..., turned:] = torch.tensor([-0.0, float("inf"), float("-inf"), 1e-7], dtype=dtype, device=dev()).repeat(d)[: d - turned]
    q[0, 0, 0, 0] = float("inf")  # one pair of one token: its two values and no others
    y, _ = cr.axial_rotary(q, None, _positions(20, axes, 52, top=7) + 1, axes, interleaved=interleaved)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(y[..., turned:].contiguous().view(bits), q[..., turned:].contiguous().view(bits))
    finite = torch.isfinite(y[..., :turned])
    assert int((~finite).sum()) == 2 and not finite[0, 0, 0, 0] and not finite[0, 0, 0, 1 if interleaved else turned // 2]


def test_positions_of_each_sample_types_and_size():
    axes, t = (16, 24, 24), 21
    q, k = randn((3, 4, t, 64), torch.float32, 11), randn((3, 2, t, 64), torch.float32, 12)
    pos = torch.stack([_positions(t, axes, 13 + i) for i in range(3)])
    for p in (pos, pos.long(), pos.int(), pos.double(), pos.transpose(0, 1).contiguous().transpose(0, 1), -pos, pos + 0.25):
        yq, yk = cr.axial_rotary(q, k, p, axes)
        assert_within(yq, *_rotate64(q, p.float(), axes, 10000.0, True))
        assert_within(yk, *_rotate64(k, p.float(), axes, 10000.0, True))
    far = pos * 1000 + 16_000_000  # positions near 2^24: the angle must still be right to 32 bits
    yq, _ = cr.axial_rotary(q, k, far, axes)
    assert_within(yq, *_rotate64(q, far, axes, 10000.0, True))


def test_turning_back_and_differences():
    axes = (16, 56, 56)
    q, pos = randn((1, 2, 30, 128), torch.float32, 21).requires_grad_(), _positions(30, axes, 22)
    y, none = cr.axial_rotary(q, None, pos, axes)
    assert none is None
    dy, v = randn(q.shape, torch.float32, 23), randn(q.shape, torch.float32, 24)
    (dq,) = torch.autograd.grad(y, q, dy)
    # linear: a difference over any step is the directional derivative, up to its float32 rounding
    d = cr.axial_rotary(q.detach() + v, None, pos, axes)[0].double() - y.detach().double()
    got, want = (dy.double() * d).sum(), (dq.double() * v.double()).sum()
    bound = 16 * U * (dy.abs().double() * (q.detach().abs() + v.abs() + 1).double()).sum() * 2
    assert (got - want).abs() <= bound
    back = torch.autograd.grad(cr.axial_rotary(q, None, pos, axes)[0], q, y.detach())[0]
    assert (back - q.detach()).abs().max() <= 40 * U * q.detach().abs().max()


def test_empty_and_missing():
    axes = (4, 4)
    q = torch.empty((2, 3, 0, 8), dtype=torch.bfloat16, device=dev(), requires_grad=True)
    y, _ = cr.axial_rotary(q, None, torch.empty((0, 2), device=dev()), axes)
    assert y.shape == q.shape and torch.autograd.grad(y.sum(), q)[0].shape == q.shape
    q, k = randn((1, 2, 4, 8), torch.float32, 1).requires_grad_(), randn((1, 2, 4, 8), torch.float32, 2)
    pos = _positions(4, axes, 3)
    yq, yk = cr.axial_rotary(q, k, pos, axes)  # only the queries want a gradient, and only the keys' is given
    (gq,) = torch.autograd.grad(yq, q, torch.ones_like(yq), retain_graph=True)
    assert_within(gq, *_rotate64(torch.ones_like(yq).detach(), pos, axes, 10000.0, True, -1.0))


def test_offsets_past_32_bits():
    axes, t, h = (32, 48, 48), 70001, 240
    pos = _positions(t, axes, 31)
    q = randn((1, t, h, 128), torch.bfloat16, 32).transpose(1, 2)
    y, _ = cr.axial_rotary(q, None, pos, axes)
    for tokens in (slice(0, 2), slice(t - 2, t)):
        w, s = _rotate64(q[:, :, tokens], pos[tokens], axes, 10000.0, True)
        assert_within(y[:, :, tokens], w, s)
    assert_no_device_error()


def test_other_stream():
    axes = (16, 56, 56)
    q, k, pos = randn((1, 4, 64, 128), torch.bfloat16, 1), randn((1, 4, 64, 128), torch.bfloat16, 2), _positions(64, axes, 3)
    want = cr.axial_rotary(q, k, pos, axes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cr.axial_rotary(q, k, pos, axes)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    q, pos = randn((1, 2, 4, 128), torch.bfloat16, 1), torch.zeros((4, 2), device=dev())
    for axes in ((), (3, 4), (0, 4), (-2, 4), (100, 100)):
        with pytest.raises(ValueError, match="axis widths"):
            cr.axial_rotary(q, None, pos, axes)
    with pytest.raises(ValueError, match="positions must be"):
        cr.axial_rotary(q, None, pos[:3], (4, 4))
    with pytest.raises(ValueError, match="do not match"):
        cr.axial_rotary(q, q[:, :, :3], pos, (4, 4))
    with pytest.raises(ValueError, match="do not match"):
        cr.axial_rotary(q, q.float(), pos, (4, 4))
    with pytest.raises(ValueError, match="theta"):
        cr.axial_rotary(q, None, pos, (4, 4), theta=0.0)
    with pytest.raises(NotImplementedError, match="head dimension"):
        cr.axial_rotary(randn((1, 1, 4, 258), torch.bfloat16, 1), None, pos, (4, 4))
    with pytest.raises(ValueError, match="CUDA"):
        cr.axial_rotary(q.cpu(), None, pos.cpu(), (4, 4))
    with pytest.raises(ValueError, match="batch, heads"):
        cr.axial_rotary(q[0], None, pos, (4, 4))
