"""The optimizer class on the device: counts in captured steps, states loaded and saved between them."""

from __future__ import annotations

import io

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import dev
from tests.ops64 import U, randn

pytestmark = pytest.mark.gpu


def _parameters(seed=1, shapes=((40, 30), (300,), (7, 9, 11))):
    return [torch.nn.Parameter(randn(s, torch.float32, seed + i)) for i, s in enumerate(shapes)]


def _set_grads(params, seed):
    for i, p in enumerate(params):
        g = randn(p.shape, p.dtype, seed + i)
        if p.grad is None:
            p.grad = g
        else:
            p.grad.copy_(g)


def _captured(optimizer):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optimizer.step()
    return graph


def test_capture_right_after_loading():
    # torch's state has no count of the group: each replay has to count on from the parameters' own
    params, eager = _parameters(), _parameters()
    theirs = torch.optim.AdamW(eager, lr=1e-2, weight_decay=0.1, capturable=True)
    for step in range(3):
        _set_grads(eager, 50 + 10 * step)
        theirs.step()
    optimizer = cr.AdamW(params)
    optimizer.load_state_dict(theirs.state_dict())
    with torch.no_grad():
        for p, q in zip(params, eager):
            p.copy_(q)
    _set_grads(params, 90)
    graph = _captured(optimizer)
    for step in range(4):
        for tensors in (params, eager):
            _set_grads(tensors, 100 + 10 * step)
        graph.replay()
        theirs.step()
        for p, q in zip(params, eager):  # the steps' own bounds: 8 U of the parameter, 64 U of updates of at most 0.1
            assert ((p - q).abs() <= (step + 1) * (8 * U * q.abs() + 64 * U * 0.1)).all()
    assert optimizer.param_groups[0]["step"].item() == 7


def test_a_capture_that_would_hold_the_count_is_refused():
    params = _parameters()
    optimizer = cr.AdamW(params)
    _set_grads(params, 10)
    optimizer.step()
    optimizer.param_groups[0]["capturable"] = True
    with pytest.raises(RuntimeError, match="before the capture"):
        _captured(optimizer)
    optimizer.step()
    graph = _captured(optimizer)
    graph.replay()
    graph.replay()
    assert optimizer.param_groups[0]["step"].item() == 4


def test_a_rate_on_the_device_after_loading_from_the_host():
    params, others = _parameters(), _parameters()
    optimizer = cr.AdamW(params, lr=torch.tensor(1e-2, device=dev()), state_bits=8, capturable=True)
    _set_grads(params, 20)
    optimizer.step()
    file = io.BytesIO()
    torch.save(optimizer.state_dict(), file)
    file.seek(0)
    state = torch.load(file, map_location="cpu", weights_only=False)
    assert state["param_groups"][0]["lr"].device.type == "cpu"
    loaded = cr.AdamW(others, state_bits=8)
    loaded.load_state_dict(state)
    with torch.no_grad():
        for p, q in zip(params, others):
            q.copy_(p)
    for tensors, o in ((params, optimizer), (others, loaded)):
        _set_grads(tensors, 30)
        o.step()
    assert loaded.param_groups[0]["lr"].device == dev()
    assert all(torch.equal(p, q) for p, q in zip(params, others))


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_and_steps_of_empty_parameters_are_clipped_too(bits):
    params, alone = _parameters(), _parameters()
    empty = [torch.nn.Parameter(torch.zeros((0, 4), device=dev()))]
    optimizer = cr.AdamW([dict(params=params), dict(params=empty)], state_bits=bits, max_norm=0.5)
    other = cr.AdamW(alone, state_bits=bits, max_norm=0.5)
    for step in range(2):
        for tensors in (params, alone, empty):
            _set_grads(tensors, 40 + step)
        optimizer.step()
        other.step()
        assert optimizer.last_norm.item() == other.last_norm.item() > 0.5
        assert all(torch.equal(p, q) for p, q in zip(params, alone))
        assert optimizer.state[params[0]]["step"] == optimizer.state[empty[0]]["step"] == step + 1
    only = cr.AdamW(empty, state_bits=bits, max_norm=0.5)
    only.step()
    assert only.last_norm.shape == () and only.last_norm.item() == 0
    p = empty[0].detach()
    assert cr.adamw_step([p], [p], [p], [p], None, 1, lr=1.0, max_norm=1.0).item() == 0
    assert cr.adamw_step([p], [p], [p], [p], None, 1, lr=1.0) is None
    with pytest.raises(ValueError, match="at least one gradient"):
        cr.adamw_step([p], [None], [p], [p], None, 1, lr=1.0, max_norm=1.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_autograd_sees_every_tensor_that_is_written(bits):
    params = _parameters()
    optimizer = cr.AdamW(params, state_bits=bits)
    _set_grads(params, 60)
    optimizer.step()
    tensors = [t for p in params for t in (p, *optimizer.state[p].values()) if torch.is_tensor(t)]
    assert len(tensors) == len(params) * (4 if bits == 8 else 3)
    before, grads = [t._version for t in tensors], [p.grad._version for p in params]
    optimizer.step()
    assert all(t._version > v for t, v in zip(tensors, before))
    assert grads == [p.grad._version for p in params]
    if bits == 32:  # a moment that a graph has saved
        x = torch.ones((40, 30), device=dev(), requires_grad=True)
        y = (x * optimizer.state[params[0]]["exp_avg"]).sum()
        optimizer.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
