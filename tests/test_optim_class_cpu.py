"""The optimizer class's own bookkeeping (no GPU needed): the step itself is a stand-in that records what it is given."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from convrot_mlx_b200 import _native


class Ops:
    """What ``AdamW`` calls of the binding."""

    def __init__(self):
        self.steps = []
        self.refusal = None

    def square_sums(self, grads):
        return torch.stack([g.double().square().sum() for g in grads])

    def adamw_step(self, params, grads, exp_avgs, exp_avg_sqs, scales, step, lr, *how):
        if self.refusal is not None:
            raise self.refusal
        self.steps.append(step.clone() if torch.is_tensor(step) else step)


@pytest.fixture
def ops(monkeypatch):
    stand_in = Ops()
    monkeypatch.setattr(_native, "ops", lambda: stand_in)
    return stand_in


def _parameters(shapes=((40, 30), (300,))):
    params = [torch.nn.Parameter(torch.zeros(s)) for s in shapes]
    for p in params:
        p.grad = torch.ones_like(p)
    return params


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_is_not_counted(ops, capturable):
    params = _parameters()
    optimizer = cr.AdamW(params, capturable=capturable)
    optimizer.step()
    ops.refusal = ValueError("refused")
    with pytest.raises(ValueError, match="refused"):
        optimizer.step()
    assert all(optimizer.state[p]["step"] == 1 for p in params)
    ops.refusal = None
    optimizer.step()
    assert [float(s) for s in ops.steps] == [1.0, 2.0] and all(optimizer.state[p]["step"] == 2 for p in params)


def _torch_state(params, steps=3, **how):
    other = torch.optim.AdamW(params, **how)
    for _ in range(steps):
        other.step()
    return other.state_dict()


def test_a_loaded_count_is_on_the_device_at_once(ops):
    # a state without the group's own count, whose next step may be a captured one
    params = _parameters()
    state = _torch_state(params)
    state["param_groups"][0]["capturable"] = True
    optimizer = cr.AdamW(params, capturable=True)
    optimizer.load_state_dict(state)
    count = optimizer.param_groups[0]["step"]
    assert count.item() == 3
    optimizer.step()
    assert optimizer.param_groups[0]["step"] is count and count.item() == 4 and ops.steps[0].item() == 4


def test_the_count_starts_at_that_of_the_parameters(ops):
    params = _parameters()
    optimizer = cr.AdamW(params)
    optimizer.step()
    params[0].grad = None
    optimizer.step()
    params[0].grad = torch.ones_like(params[0])
    optimizer.param_groups[0]["capturable"] = True
    optimizer.step()  # the group has taken two steps, its first parameter one
    assert optimizer.param_groups[0]["step"].item() == 3


def _loads_nothing(optimizer, state, match):
    params = optimizer.param_groups[0]["params"]
    kept = {p: {k: v.clone() if torch.is_tensor(v) else v for k, v in optimizer.state[p].items()} for p in params}
    with pytest.raises(ValueError, match=match):
        optimizer.load_state_dict(state)
    for p in params:
        now = optimizer.state[p]
        assert now.keys() == kept[p].keys()
        assert all(torch.equal(v, now[k]) if torch.is_tensor(v) else v == now[k] for k, v in kept[p].items())


@pytest.mark.parametrize("shape", [(1,), (30,), (40, 1), (30, 40), (1200,), (2, 40, 30)])
@pytest.mark.parametrize("name", ["exp_avg", "exp_avg_sq"])
@pytest.mark.parametrize("of", [0, 1])
def test_moments_of_other_shapes_are_not_loaded(ops, of, name, shape):
    # also those that would be broadcast, and those of the last parameter
    params = _parameters(((40, 30), (40, 30)))
    state = _torch_state(params)
    state["state"][of][name] = torch.ones(shape)
    optimizer = cr.AdamW(params)
    optimizer.step()
    _loads_nothing(optimizer, state, "shape")


def test_states_of_other_rules_are_not_loaded(ops):
    params = _parameters()
    other = torch.optim.SGD(params, lr=0.1, momentum=0.9)
    other.step()
    optimizer = cr.AdamW(params)
    optimizer.step()
    _loads_nothing(optimizer, other.state_dict(), "exp_avg")
    state = _torch_state(params)
    del state["state"][1]["step"]
    _loads_nothing(optimizer, state, "step")


def test_8_bit_states_are_checked_whole(ops):
    params = _parameters()
    optimizer = cr.AdamW(params, state_bits=8)
    optimizer.step()

    def changed(name, value):
        state = optimizer.state_dict()
        state["state"] = {k: dict(v) for k, v in state["state"].items()}
        state["state"][1][name] = value
        return state

    codes = torch.zeros(300, dtype=torch.uint8).view(torch.float8_e4m3fn)
    for name in ("exp_avg", "exp_avg_sq"):
        _loads_nothing(optimizer, changed(name, codes[:299]), "shape or memory layout")
        _loads_nothing(optimizer, changed(name, torch.zeros(600, dtype=torch.uint8).view(torch.float8_e4m3fn)[::2]), "layout")
    for shape in ((1, 2), (2,), (2, 1), (300, 2)):
        _loads_nothing(optimizer, changed("scales", torch.ones(shape)), "scales of shape")
    optimizer.load_state_dict(changed("scales", torch.full((2, 2), 3.0)))
    assert optimizer.state[params[1]]["scales"].eq(3).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_loading_heeds_the_hooks(ops, bits):
    params = _parameters()
    optimizer = cr.AdamW(params, state_bits=bits)
    optimizer.step()
    saved = optimizer.state_dict()
    seen = []

    def twice(_, state):  # counts changed on the way in, in a dictionary of the hook's own
        return {**state, "state": {k: {**v, "step": 2 * v["step"]} for k, v in state["state"].items()}}

    def look(o):
        seen.append({k: v if k == "step" else v.dtype for k, v in o.state[params[0]].items()})

    hooks = [optimizer.register_load_state_dict_pre_hook(twice), optimizer.register_load_state_dict_post_hook(look)]
    optimizer.load_state_dict(saved)
    kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
    want = {"step": 2, "exp_avg": kind, "exp_avg_sq": kind, **({"scales": torch.float32} if bits == 8 else {})}
    assert seen == [want] and all(optimizer.state[p]["step"] == 2 for p in params)
    assert all(v["step"] == 1 for v in saved["state"].values())
    for hook in hooks:
        hook.remove()
    optimizer.load_state_dict(saved)  # and the class leaves none of its own
    assert optimizer.state[params[0]]["step"] == 1 and len(seen) == 1
    with pytest.raises(ValueError, match="different"):
        optimizer.load_state_dict({**saved, "param_groups": saved["param_groups"] * 2})
    assert optimizer.state[params[0]]["step"] == 1


def test_loading_keeps_no_copy_in_another_type(ops):
    # 8-bit moments of a float32 parameter are loaded as they are: no tensor of four times their size on the way
    params = _parameters(((1 << 16,),))
    optimizer = cr.AdamW(params, state_bits=8)
    optimizer.step()
    saved = optimizer.state_dict()
    with torch.profiler.profile(profile_memory=True) as profile:
        optimizer.load_state_dict(saved)
    largest = max(event.self_cpu_memory_usage for event in profile.events())
    assert largest < 4 * (1 << 16), largest


def test_a_group_without_parameters_is_loaded(ops):
    params = _parameters()
    optimizer = cr.AdamW([dict(params=params), dict(params=[])], lr=torch.tensor(1e-2))
    optimizer.step()
    optimizer.load_state_dict(optimizer.state_dict())
    assert optimizer.state[params[0]]["step"] == 1 and optimizer.param_groups[0]["lr"].item() == torch.tensor(1e-2).item()


def test_counts_of_replays_are_saved(ops):
    params = _parameters()
    optimizer = cr.AdamW(params, capturable=True)
    optimizer.step()
    optimizer.param_groups[0]["step"].add_(6.0)  # as six replays of a captured step do
    state = optimizer.state_dict()
    assert [v["step"] for v in state["state"].values()] == [7, 7] and state["param_groups"][0]["step"].item() == 7
    other = torch.optim.AdamW(params)  # whose steps would be corrected for it
    state["param_groups"][0]["capturable"] = False
    other.load_state_dict(state)
    assert all(int(other.state[p]["step"]) == 7 for p in params)


def test_the_count_goes_back_to_the_parameters(ops):
    params = _parameters()
    optimizer = cr.AdamW(params, capturable=True)
    optimizer.step()
    optimizer.param_groups[0]["step"].add_(6.0)
    optimizer.param_groups[0]["capturable"] = False
    optimizer.step()
    assert ops.steps[-1] == 8 and optimizer.state[params[0]]["step"] == 8
    optimizer.param_groups[0]["capturable"] = True
    optimizer.step()
    assert ops.steps[-1].item() == 9
