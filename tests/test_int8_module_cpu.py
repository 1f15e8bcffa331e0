"""Int8Linear keeps its scales and bias in float32 under casts and moves of the module (no GPU needed)."""

from __future__ import annotations

import copy

import pytest
import torch

import convrot_mlx_b200 as cr


def _layer(bias=True):
    layer = cr.Int8Linear(20, 6, bias=bias)
    layer.qweight.random_(-127, 128)
    layer.scales.copy_(torch.rand(6) * 1e-3 + 1e-4)
    if bias:
        layer.bias.copy_(torch.randn(6))
    return layer


CASTS = {
    "bfloat16": lambda m: m.to(torch.bfloat16),
    "half": lambda m: m.half(),
    "double": lambda m: m.double(),
    "cpu, float16": lambda m: m.to("cpu", torch.float16),
    "there and back": lambda m: m.bfloat16().float(),
    "of a model": lambda m: torch.nn.Sequential(torch.nn.Linear(4, 4), m).to(torch.bfloat16)[1],
    "a copy": lambda m: copy.deepcopy(m).half(),
}


@pytest.mark.parametrize("cast", CASTS.values(), ids=CASTS)
@pytest.mark.parametrize("bias", [True, False])
def test_values_survive_casts(cast, bias):
    layer = _layer(bias)
    want = {k: v.clone() for k, v in layer.state_dict().items()}
    got = cast(layer).state_dict()
    assert got.keys() == want.keys()
    for name, value in want.items():
        assert got[name].dtype == value.dtype and torch.equal(got[name], value), name


def test_moves_still_move():
    layer = _layer().to("meta")
    assert all(b.is_meta for b in layer.buffers())
    empty = cr.Int8Linear(20, 6, device="meta").to(torch.bfloat16).to_empty(device="cpu")
    assert empty.scales.dtype == empty.bias.dtype == torch.float32 and empty.scales.device.type == "cpu"
    empty.load_state_dict(_layer().state_dict())
    moved = _layer().to("meta", torch.bfloat16)
    assert moved.scales.is_meta and moved.scales.dtype == torch.float32
