"""The AdamW step over many tensors at once, with its moments in 32 bits or in 8, and the gradient norm that clips it.

What is trained around frozen quantized linears (modulations, norms, adapters)
is many tensors, often small, and for a whole block its moments are the largest
part of what training holds.  One launch updates up to 512 tensors; the norm
stays on the device, and the step scales the gradients by it as it reads them.
No counterpart in the reference (it does not train).

Moments in 8 bits: m and sqrt(v) as float8_e4m3fn with a float32 scale each for
256 consecutive values of a tensor (the largest becomes 448).  A block whose
scales are not finite, as an infinite or NaN gradient makes them, stays NaN.
They are rounded to nearest, 2^-4 of a value at most, so a value keeps its code
where a step changes it by less: sqrt(v), which a step without a gradient lowers
by (1 - b2) / 2, follows its average for b2 up to 0.95 only.  Where the gradients
of a quarter of a block's values become four times smaller, their median root is
1.9 times too large 200 steps later at b2 0.98 (right after 1500), 2.2 at 0.99
(2.9 after 1500), 1.4 at 0.999 (1.9); where they become four times larger, that
of the others is 1.24 times too large at 0.99 and 1.44 at 0.999.  Steps are too
short by as much.
"""

from __future__ import annotations

import itertools
from typing import Iterable, Sequence

import torch

from . import _native

MOMENT_BLOCK = 256  # values of a tensor whose 8-bit moments share their scales


def grad_norm(grads: Iterable[torch.Tensor | None]) -> torch.Tensor:
    """The 2-norm of all values of ``grads`` (CUDA tensors of one device; None is passed over), float32 on the device.

    Squares are summed in 64 bits, so neither large nor small values leave its
    range before the norm itself does; the same bits on every call."""

    return _native.ops().grad_norm(grads if isinstance(grads, (list, tuple)) else list(grads))


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor | None], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], scales: Sequence[torch.Tensor] | None, step, *, lr, betas=(0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, max_norm: float | None = None) -> torch.Tensor | None:
    """One AdamW step in place: parameters float32, float16 or bfloat16 with gradients of their type (None: left as it is).

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
        p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v / (1 - b2^step)) + eps)

    ``scales`` None: ``exp_avgs`` and ``exp_avg_sqs`` hold m and v in float32.
    Else they hold float8_e4m3fn codes of m and of sqrt(v), and ``scales`` for
    each parameter (ceil(n / 256), 2) float32, the scales of both for each 256
    values; zeros are the start of either.  ``step`` counts from 1; ``step`` and ``lr``
    may each be one float32 on the device, which a captured step reads when
    it is replayed.  ``max_norm``: gradients are scaled by
    min(1, max_norm / (norm + 1e-6)) as they are read, with the norm of them all, which
    is returned.  Gradients are not changed.  A parameter that is not contiguous has to be dense, with
    its moments laid out as it is.  Parameters, moments and scales may not overlap one another or another's gradient."""

    return _native.ops().adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales, step, lr, betas[0], betas[1], eps,
                                    weight_decay, max_norm, None)


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.shape == b.shape and all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


class AdamW(torch.optim.Optimizer):
    """AdamW by ``adamw_step``: all parameters of a group in one launch.

    ``state_bits`` 8 keeps the moments in 8 bits (2.03 bytes a parameter; with
    ``betas[1]`` up to 0.95, not its default: above, roots lag behind as this module's text
    says), 32 in float32 (8 bytes) whatever the parameter's type, under the names of
    ``torch.optim.AdamW``, whose state dict can be loaded.  ``max_norm`` clips by
    the norm of all gradients of all groups; ``last_norm`` is that of the last step, on
    the device.  ``capturable``: the step count of a group is on the device
    (``group["step"]``), so that a graph that captured ``step`` counts on as it
    is replayed; all its parameters share it, and ``load_state_dict`` takes it from
    the state, as all options of a group.  ``lr`` may be one float32 on the
    device.  All parameters lie on one CUDA device."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, max_norm: float | None = None, capturable: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"moments are kept in 8 or 32 bits, not {state_bits}")
        if not torch.is_tensor(lr) and not lr >= 0:
            raise ValueError(f"the learning rate must be non-negative, got {lr}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError("eps and weight decay must be non-negative")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"the largest norm must be non-negative, got {max_norm}")
        self.state_bits = state_bits
        self.max_norm = max_norm
        self.last_norm: torch.Tensor | None = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, capturable=capturable))

    def __getstate__(self) -> dict:  # of copies and saved optimizers
        return {**super().__getstate__(), "state_bits": self.state_bits, "max_norm": self.max_norm, "last_norm": None}

    def _start(self, p: torch.Tensor) -> dict:
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW starts its moments in its first step: take one before the capture")
        keep = torch.preserve_format
        kind = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        state = self.state[p]
        state["step"] = 0
        state["exp_avg"] = torch.zeros_like(p, dtype=kind, memory_format=keep)
        state["exp_avg_sq"] = torch.zeros_like(p, dtype=kind, memory_format=keep)
        if self.state_bits == 8:
            state["scales"] = torch.zeros((-(-p.numel() // MOMENT_BLOCK), 2), dtype=torch.float32, device=p.device)
        return state

    def _put_count_on_device(self, group: dict) -> None:
        started = [p for p in group["params"] if self.state.get(p)]
        if started[0].is_cuda and torch.cuda.is_current_stream_capturing():  # each replay would set the count again
            raise RuntimeError("AdamW puts its count on the device in a step of its own: take one before the capture")
        count = max(self.state[p]["step"] for p in started)
        group["step"] = torch.full((), float(count), device=started[0].device)

    @torch.no_grad()
    def step(self, closure=None):
        """One step; returns the closure's loss, if there is one."""

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ops, sums, norm = _native.ops(), None, None
        if self.max_norm is not None:
            grads = [p.grad for group in self.param_groups for p in group["params"] if p.grad is not None]
            if not grads:
                return loss
            sums = ops.square_sums(grads)
        for group in self.param_groups:
            if not group["capturable"] and torch.is_tensor(group.get("step")):  # it was until now
                self._read_counts(group)
                del group["step"]
            capturable = group["capturable"]
            runs: dict = {}  # the parameters by their step, nearly always one
            for p in group["params"]:
                if p.grad is not None:
                    if not runs and not capturable and p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("a captured AdamW step needs capturable=True: its count has to be on the device")
                    state = self.state[p] or self._start(p)
                    runs.setdefault(0 if capturable else state["step"] + 1, []).append((p, state))
            if runs and capturable:
                if not torch.is_tensor(group.get("step")):
                    self._put_count_on_device(group)
                group["step"].add_(1.0)
            for step, run in runs.items():
                states = [state for _, state in run]
                try:
                    norm = ops.adamw_step([p for p, _ in run], [p.grad for p, _ in run], [s["exp_avg"] for s in states],
                                          [s["exp_avg_sq"] for s in states],
                                          [s["scales"] for s in states] if self.state_bits == 8 else None,
                                          group["step"] if capturable else step, group["lr"], *group["betas"],
                                          group["eps"], group["weight_decay"], self.max_norm, sums)
                except (ValueError, NotImplementedError):  # refused: not a step
                    if capturable:
                        group["step"].sub_(1.0)
                    raise
                for state in states:
                    state["step"] += 1
        self.last_norm = norm
        return loss

    def _read_counts(self, group: dict) -> None:
        """The count on the device, which replays of a captured step advance, as that of the group's parameters."""

        count = int(group["step"].item())
        for p in group["params"]:
            if self.state.get(p):
                self.state[p]["step"] = count

    def state_dict(self) -> dict:
        """The state, under the names of ``torch.optim.AdamW``; counts that are on the device are read back."""

        for group in self.param_groups:
            if torch.is_tensor(group.get("step")):
                self._read_counts(group)
        return super().state_dict()

    def load_state_dict(self, state_dict: dict) -> None:
        """Load a state of this class, or with ``state_bits`` 32 of ``torch.optim.AdamW``; moments keep their types."""

        # The state is taken as the pre-hooks leave it, and in place before any post-hook.  The base class loads the
        # groups alone: it would cast the moments to the parameters' type.
        loaded: list = []

        def check(_, state: dict) -> dict:
            loaded.extend(self._checked(state))
            ids = {key for group in state["param_groups"] for key in group["params"]}
            return {**state, "state": {key: rest for key, rest in state["state"].items() if key not in ids}}

        before = self.register_load_state_dict_pre_hook(check)
        after = self.register_load_state_dict_post_hook(lambda _: self._load(loaded), prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            before.remove()
            after.remove()

    def _checked(self, state_dict: dict) -> list:
        """The parameters that have a state in ``state_dict``, each with it; refused as a whole."""

        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("this AdamW has neither amsgrad nor maximize")
            if group.get("decoupled_weight_decay") is False and group["weight_decay"] != 0:
                raise ValueError("this AdamW's weight decay is decoupled, that of the state is not")
        ids = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        params = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        loaded = [(p, state_dict["state"][key]) for key, p in zip(ids, params) if state_dict["state"].get(key)]
        for p, saved in loaded:
            if ("scales" in saved) != (self.state_bits == 8):
                raise ValueError(f"the state's moments are not kept in {self.state_bits} bits")
            if "step" not in saved or not all(torch.is_tensor(saved.get(name)) for name in ("exp_avg", "exp_avg_sq")):
                raise ValueError(f"the state has no step, exp_avg and exp_avg_sq, but {sorted(saved)}")
            for moment in (saved["exp_avg"], saved["exp_avg_sq"]):
                if self.state_bits == 8 and not _same_layout(moment, p):
                    raise ValueError("8-bit moments were kept for a parameter of another shape or memory layout")
                if moment.shape != p.shape:
                    raise ValueError(f"moments of shape {tuple(moment.shape)} are not those of a parameter of shape {tuple(p.shape)}")
            if self.state_bits == 8 and tuple(saved["scales"].shape) != (-(-p.numel() // MOMENT_BLOCK), 2):
                raise ValueError(f"scales of shape {tuple(saved['scales'].shape)} are not those of {p.numel()} 8-bit moments")
        return loaded

    @torch.no_grad()
    def _load(self, loaded: list) -> None:
        kind = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        for p, saved in loaded:
            state = {"step": int(saved["step"])}
            for name in ("exp_avg", "exp_avg_sq"):
                # the parameter's own layout, whatever that of the saved tensor was
                state[name] = torch.empty_like(p, dtype=kind, memory_format=torch.preserve_format).copy_(saved[name])
            if self.state_bits == 8:
                state["scales"] = saved["scales"].to(p.device, torch.float32, copy=True).contiguous()
            self.state[p] = state
        for group in self.param_groups:
            group.setdefault("capturable", False)
            if not group["params"]:
                continue
            if torch.is_tensor(group["lr"]):  # wherever the state was kept
                group["lr"] = group["lr"].to(group["params"][0].device, torch.float32, copy=True)
            if torch.is_tensor(group.get("step")):
                group["step"] = group["step"].to(group["params"][0].device, torch.float32, copy=True)
            elif group["capturable"] and any(self.state.get(p) for p in group["params"]):
                self._put_count_on_device(group)
