"""The 8-bit and training operators together in a block (dit_finetune.py): its output and gradients against the same
block in torch's own operators with the dequantized weights, and a short training run.

Tolerance: activations, their gradients and the saved GELU input are held in 8 bits (steps of 1/127 of a token's or
group's largest magnitude, about 3 to 4 standard deviations: 0.7% to 0.9% noise for each of the quantized tensors on a
path) and everything else in bfloat16 (0.2% a rounding): a few percent in the 2-norm through the block, 8% taken as
the bound."""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

import convrot_mlx_b200 as cr
import dit_finetune as ft
from tests.gpu_util import assert_no_device_error, dev

pytestmark = pytest.mark.gpu


class DenseLinear(torch.nn.Module):
    """The dequantized form of a frozen 8-bit linear."""

    def __init__(self, q: cr.Int8Linear):
        super().__init__()
        self.weight = q.qweight[:, :q.in_features].float() * q.scales[:, None]
        self.bias = q.bias

    def forward(self, x):
        return F.linear(x, self.weight, self.bias)


def _reference_forward(block, x, vec, positions):
    """Block.forward in torch operators and float32."""

    s1, c1, g1, s2, c2, g2 = block.modulation(F.silu(vec)).unsqueeze(1).chunk(6, dim=-1)
    norm = lambda t, s, c: F.layer_norm(t, t.shape[-1:], eps=1e-6) * (1 + c) + s  # noqa: E731
    q, k, v = block.qkv(norm(x, s1, c1)).unflatten(-1, (3, block.heads, -1)).unbind(2)
    q = F.layer_norm(q, q.shape[-1:], block.q_norm.weight, block.q_norm.bias, 1e-6).transpose(1, 2)
    k = F.layer_norm(k, k.shape[-1:], block.k_norm.weight, block.k_norm.bias, 1e-6).transpose(1, 2)
    ang = torch.cat([positions[:, a, None] * 10000.0 ** (-torch.arange(0, w, 2, device=dev()).float() / w)
                     for a, w in enumerate(block.axes)], -1)
    turn = torch.polar(torch.ones_like(ang), ang)
    rot = lambda t: torch.view_as_real(torch.view_as_complex(t.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)  # noqa: E731
    a = F.scaled_dot_product_attention(rot(q), rot(k), v.transpose(1, 2)).transpose(1, 2).flatten(2)
    x = x + g1 * block.proj(a)
    return x + g2 * block.down(F.gelu(block.up(norm(x, s2, c2)), approximate="tanh"))


def test_block_against_torch():
    block = ft.build(768, 12, dev(), seed=3)
    dense = copy.deepcopy(block).float()
    for name in ft.FROZEN:
        setattr(dense, name, DenseLinear(getattr(block, name)))
    g = torch.Generator(device=dev()).manual_seed(4)
    positions = ft.grid_positions(2, 5, 7, dev())
    x = torch.randn((2, 70, 768), generator=g, device=dev()).bfloat16().requires_grad_()
    vec = torch.randn((2, 768), generator=g, device=dev()).bfloat16()
    dy = torch.randn((2, 70, 768), generator=g, device=dev()).bfloat16()
    x32 = x.detach().float().requires_grad_()
    y = block(x, vec, positions)
    y32 = _reference_forward(dense, x32, vec.float(), positions)
    rel = lambda a, b: ((a.float() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(y, y32) < 0.08
    params = [n for n, _ in block.named_parameters()]
    assert set(params) == {"modulation.weight", "modulation.bias", "q_norm.weight", "q_norm.bias", "k_norm.weight",
                           "k_norm.bias"}
    got = torch.autograd.grad(y, [x, *block.parameters()], dy)
    want = torch.autograd.grad(y32, [x32, *dense.parameters()], dy.float())
    for name, a, b in zip(["x", *params], got, want):
        assert a.shape == b.shape
        if name == "k_norm.bias":  # moves every key of a head nearly alike: close to nothing survives the softmax
            continue
        assert rel(a, b) < 0.08, (name, rel(a, b))
    assert_no_device_error()


def test_training_lowers_the_loss_and_repeats():
    losses = ft.train(12, 768, 12, 2, 2, 6, 8)
    assert losses[-1] < 0.7 * losses[0]
    assert all(b < a * 1.05 for a, b in zip(losses, losses[1:]))
