"""The 8-bit floating-point linears, the gradient norm and AdamW together in a training step (dit_finetune.py): the
block's output and gradients against the same block in torch's own operators with the dequantized weights, and a step
of both optimizers from these gradients.

Tolerance: activations and their gradients are held in e4m3 (2^-4 of a value at most, 2.6% on average) in each of the
four projections on a path, everything else in bfloat16 (0.2% a rounding): about 2.6% times the square root of 8, 12%
taken as the bound."""

from __future__ import annotations

import copy
import math

import pytest
import torch
import torch.nn.functional as F

import convrot_mlx_b200 as cr
import dit_finetune as ft
from tests.fp8_64 import values_of_blocks
from tests.gpu_util import assert_no_device_error, dev
from tests.test_gpu_finetune import _reference_forward

pytestmark = pytest.mark.gpu


class DenseLinear(torch.nn.Module):
    """The dequantized form of a frozen 8-bit floating-point linear."""

    def __init__(self, q: cr.Fp8Linear):
        super().__init__()
        codes = q.qweight.view(torch.float8_e4m3fn)[:, :q.in_features]
        self.weight = values_of_blocks(codes, q.scales.view(torch.float8_e8m0fnu)).float()
        self.bias = q.bias

    def forward(self, x):
        return F.linear(x, self.weight, self.bias)


def _setup():
    block = ft.build(768, 12, dev(), seed=3, linears="fp8")
    g = torch.Generator(device=dev()).manual_seed(4)
    x = torch.randn((2, 70, 768), generator=g, device=dev()).bfloat16().requires_grad_()
    vec = torch.randn((2, 768), generator=g, device=dev()).bfloat16()
    dy = torch.randn((2, 70, 768), generator=g, device=dev()).bfloat16()
    return block, x, vec, dy, ft.grid_positions(2, 5, 7, dev())


def test_block_against_torch():
    block, x, vec, dy, positions = _setup()
    dense = copy.deepcopy(block).float()
    for name in ft.FROZEN:
        setattr(dense, name, DenseLinear(getattr(block, name)))
    x32 = x.detach().float().requires_grad_()
    y, y32 = block(x, vec, positions), _reference_forward(dense, x32, vec.float(), positions)
    rel = lambda a, b: ((a.float() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(y, y32) < 0.12
    params = [n for n, _ in block.named_parameters()]
    got = torch.autograd.grad(y, [x, *block.parameters()], dy)
    want = torch.autograd.grad(y32, [x32, *dense.parameters()], dy.float())
    for name, a, b in zip(["x", *params], got, want):
        assert a.shape == b.shape
        if name == "k_norm.bias":  # moves every key of a head nearly alike: close to nothing survives the softmax
            continue
        assert rel(a, b) < 0.12, (name, rel(a, b))
    assert_no_device_error()


@pytest.mark.parametrize("bits", [32, 8])
def test_step_from_the_block_s_gradients(bits):
    block, x, vec, dy, positions = _setup()
    params = list(block.parameters())
    grads = torch.autograd.grad(block(x, vec, positions), params, dy)
    before = [p.detach().clone() for p in params]
    for p, g in zip(params, grads):
        p.grad = g
    optimizer = cr.AdamW(params, lr=1e-2, weight_decay=0.0, state_bits=bits, max_norm=1.0)
    optimizer.step()
    exact = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    assert abs(optimizer.last_norm.item() - exact) <= 1e-6 * exact
    factor = min(1.0, 1.0 / (exact + 1e-6))
    for p, b, g in zip(params, before, grads):  # the first step: m / sqrt(v) is g / |g| but for eps
        g64 = g.double() * factor
        want = b.double() - 1e-2 * g64 / (g64.abs() + 1e-8)
        assert ((p.double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-2 * 2.0 ** -8 + 1e-7).all()


def test_captured_training_step():
    """Forward, backward, norm and step in one graph, replayed twice, against the same steps without a graph."""

    states = []
    for captured in (True, False):
        block, x, vec, dy, positions = _setup()
        params = list(block.parameters())
        optimizer = cr.AdamW(params, lr=1e-3, state_bits=8, max_norm=1.0, capturable=captured)

        def step():
            for p, g in zip(params, torch.autograd.grad(block(x, vec, positions), params, dy)):
                p.grad.copy_(g)
            optimizer.step()

        for p in params:
            p.grad = torch.zeros_like(p)
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            graph.replay()
            graph.replay()
        else:
            for _ in range(3):
                step()
        states.append([p.detach().clone() for p in params])
    for a, b in zip(*states):  # three updates of at most 1e-3 * 10, each a bfloat16 rounding apart at most
        assert ((a.float() - b.float()).abs() <= 3 * (b.float().abs() * 2.0 ** -7 + 1e-3 * 2.0 ** -7)).all()
    assert_no_device_error()


@pytest.mark.parametrize("linears", ["int8", "fp8"])
@pytest.mark.parametrize("optimizer", ["adam", "adamw32", "adamw8"])
def test_example_runs(linears, optimizer):
    losses = ft.train(3, 768, 12, 1, 2, 3, 4, linears=linears, optimizer=optimizer)
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses)
