"""Frozen 8-bit weights under hooks of saved tensors, which may give them back laid out in another way."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import assert_no_device_error
from tests.ops64 import DTYPES, randn

pytestmark = pytest.mark.gpu

OPS = {"fp8": (cr.fp8_linear, cr.quantize_fp8_weight), "int8": (cr.int8_linear, cr.quantize_int8_weight)}


def _apart(t):  # the same values, every stride doubled and the start off any boundary
    wide = torch.empty([2 * s + 1 for s in t.shape], dtype=t.dtype, device=t.device)
    view = wide[tuple(slice(1, None, 2) for _ in t.shape)]
    view.copy_(t)
    return view


HOOKS = {
    "host": torch.autograd.graph.save_on_cpu,
    "pinned host": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    "packed": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)),
    "apart": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, _apart),
}


@pytest.mark.parametrize("hook", list(HOOKS))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("op", list(OPS))
@pytest.mark.parametrize("m,k,n", [(1, 203, 48), (7, 80, 48), (40, 203, 300), (300, 1301, 520)])
def test_gradient_of_a_weight_that_was_moved(op, m, k, n, dtype, hook):
    linear, quantize = OPS[op]
    w, ws = quantize(randn((n, k), torch.float32, 1))
    x, dy = randn((m, k), dtype, 2).requires_grad_(), randn((m, n), dtype, 3)
    (want,) = torch.autograd.grad(linear(x, w, ws), x, dy)
    with HOOKS[hook]():
        y = linear(x, w, ws)
    for _ in range(2):
        (dx,) = torch.autograd.grad(y, x, dy, retain_graph=True)
        assert torch.equal(dx, want)
    assert_no_device_error()


@pytest.mark.parametrize("hook", list(HOOKS))
def test_int8_gradient_in_ranges_of_a_weight_that_was_moved(hook):
    n, k = 131100, 35
    w, ws = cr.quantize_int8_weight(randn((n, k), torch.float32, 11))
    x, dy = randn((9, k), torch.bfloat16, 12).requires_grad_(), randn((9, n), torch.bfloat16, 13)
    (want,) = torch.autograd.grad(cr.int8_linear(x, w, ws), x, dy)
    with HOOKS[hook]():
        y = cr.int8_linear(x, w, ws)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
