"""Norm, rotary and saved-8-bit GELU under hooks of saved tensors, which may give them back laid out in another way."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import dev
from tests.ops64 import DTYPES, randn
from tests.test_gpu_saved_weights import HOOKS

pytestmark = pytest.mark.gpu


def _same_gradients(call, inputs, seed, hook):
    dy = randn(call().shape, inputs[0].dtype, seed)
    want = torch.autograd.grad(call(), inputs, dy)
    with HOOKS[hook]():
        y = call()
    got = torch.autograd.grad(y, inputs, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("hook", list(HOOKS))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", [(1, 5), (33, 300), (200, 768)])
def test_norm(dtype, rows, features, hook):
    x = randn((rows, features), dtype, 1).requires_grad_()
    w, b = randn((features,), dtype, 2).requires_grad_(), randn((features,), dtype, 3).requires_grad_()
    _same_gradients(lambda: cr.layer_norm(x, w, b), [x, w, b], 4, hook)
    # vectors of each sample, columns of one projection's output
    x3 = randn((3, rows, features), dtype, 5).requires_grad_()
    vectors = randn((3, 6 * features), dtype, 6).requires_grad_()

    def call():
        shift, scale = vectors.chunk(6, dim=-1)[1:3]
        return cr.modulated_layer_norm(x3, shift, scale)

    _same_gradients(call, [x3, vectors], 7, hook)


@pytest.mark.parametrize("hook", list(HOOKS))
@pytest.mark.parametrize("batched", [False, True])
def test_rotary(batched, hook):
    q, k = (randn((2, 3, 30, 64), torch.bfloat16, i).requires_grad_() for i in (1, 2))
    positions = torch.randint(0, 50, (2, 30, 2) if batched else (30, 2), device=dev(),
                              generator=torch.Generator(device=dev()).manual_seed(3)).float()
    _same_gradients(lambda: torch.cat(cr.axial_rotary(q, k, positions, (16, 32))), [q, k], 4, hook)


@pytest.mark.parametrize("hook", list(HOOKS))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", [(1, 1), (7, 130), (100, 1024)])
def test_gelu(dtype, rows, features, hook):
    x = randn((rows, features), dtype, 1).requires_grad_()
    _same_gradients(lambda: cr.gelu_tanh_saved8(x), [x], 2, hook)


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_gelu_saved_in_a_pool_of_bytes(offset):
    x = randn((9, 300), torch.bfloat16, 1).requires_grad_()
    dy = randn(x.shape, torch.bfloat16, 2)
    (want,) = torch.autograd.grad(cr.gelu_tanh_saved8(x), x, dy)

    def unpack(t):
        pool = torch.zeros(t.numel() + 16, dtype=t.dtype, device=t.device)
        pool[offset:offset + t.numel()] = t
        return pool[offset:offset + t.numel()]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = cr.gelu_tanh_saved8(x)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
