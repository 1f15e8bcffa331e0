"""float32 outputs of the 8-bit floating-point product over many channels: sums in ranges of 8192, by either entry point."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.fp8_64 import product64, values_of_blocks, values_of_rows
from tests.gpu_util import assert_no_device_error
from tests.ops64 import DTYPES, assert_within, randn

pytestmark = pytest.mark.gpu

RANGE = 8192
# of every kernel: up to 8 tokens, few tokens with K split and not, many; odd channels
SIZES = [(1, 15360, 40), (3, 20000, 33), (5, 17000, 130), (8, 8193, 70), (8, 24576, 16), (16, 15360, 96), (40, 8320, 300),
         (100, 20000, 259), (300, 16384, 5001), (1300, 8200, 1211), (1500, 15360, 2048), (2100, 9000, 130)]


def _operands(m, k, n, seed):
    x, w = randn((m, k), torch.float32, seed), randn((n, k), torch.float32, seed + 1, 0.05)
    return x, *cr.quantize_fp8_blockwise(x), *cr.quantize_fp8_weight(w), randn((n,), torch.float32, seed + 2)


def _one_launch(m, k):
    """Whether the kernel for few tokens holds them, which needs no ranges."""

    return m <= 8 and m * (2 * k + 2 * 128 + 16 + 4 * (k // 128 + 1)) <= 96 * 1024


@pytest.mark.parametrize("m,k,n", SIZES)
def test_both_entry_points_are_the_same_sum(m, k, n):
    x, codes, xs, w, ws, bias = _operands(m, k, n, 1)
    y = cr.fp8_matmul(codes, w, xs, ws, bias, output_dtype=torch.float32)
    assert torch.equal(y, cr.fp8_linear(x, w, ws, bias))
    assert_within(y, *product64(values_of_rows(codes, xs), values_of_blocks(w, ws), bias), f"{m} {k} {n}")
    assert_no_device_error()


@pytest.mark.parametrize("m,k,n", SIZES)
def test_ranges_are_added_in_order(m, k, n):
    _, codes, xs, w, ws, bias = _operands(m, k, n, 11)
    if _one_launch(m, k):
        pytest.skip("one launch")
    want = None
    for at in range(0, k, RANGE):
        to = min(k, at + RANGE)
        spans = slice(at // 128, -(-to // 128))
        part = cr.fp8_matmul(codes[:, at:to], w[:, at:to], xs[:, spans], ws[:, spans], bias if at == 0 else None,
                             output_dtype=torch.float32)
        want = part if want is None else want + part
    assert torch.equal(cr.fp8_matmul(codes, w, xs, ws, bias, output_dtype=torch.float32), want)


@pytest.mark.parametrize("m,n", [(3, 20000), (40, 8320), (300, 16384), (1500, 15361)])
def test_gradient_over_many_channels(m, n):
    k = 200
    w, ws = cr.quantize_fp8_weight(randn((n, k), torch.float32, 21, 0.05))
    x, dy = randn((m, k), torch.float32, 22).requires_grad_(), randn((m, n), torch.float32, 23)
    (dx,) = torch.autograd.grad(cr.fp8_linear(x, w, ws), x, dy)
    codes, scales = cr.quantize_fp8_blockwise(dy)
    # the same matrix, laid out the other way: its blocks are square, so codes and scales are turned with it
    turned = cr.fp8_matmul(codes, w.t().contiguous(), scales, ws.t().contiguous(), output_dtype=torch.float32)
    assert_within(dx, *product64(values_of_rows(codes, scales), values_of_blocks(w, ws).T))
    off = (dx - turned).norm() / turned.norm()
    assert off <= 2.0 ** -20  # two such sums, 2^-21 of the norm each


@pytest.mark.parametrize("dtype", DTYPES)
def test_outputs_are_written_whatever_was_there(dtype):
    # the first range does not add: an output in memory that held something else
    m, k, n = 130, 20000, 264
    x, codes, xs, w, ws, bias = _operands(m, k, n, 31)
    want = cr.fp8_matmul(codes, w, xs, ws, bias, output_dtype=dtype)
    for _ in range(3):
        junk = [torch.full((m, n), float("nan"), dtype=dtype, device=x.device) for _ in range(4)]
        del junk
        assert torch.equal(cr.fp8_matmul(codes, w, xs, ws, bias, output_dtype=dtype), want)


def test_captured_on_another_stream():
    m, k, n = 64, 17000, 520
    x, codes, xs, w, ws, bias = _operands(m, k, n, 41)
    want = cr.fp8_linear(x, w, ws, bias)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cr.fp8_linear(x, w, ws, bias)
        z = cr.fp8_matmul(codes, w, xs, ws, bias, output_dtype=torch.float32)
    for _ in range(3):
        y.fill_(float("nan"))
        z.fill_(float("nan"))
        graph.replay()
        assert torch.equal(y, want) and torch.equal(z, want)
    assert_no_device_error()
