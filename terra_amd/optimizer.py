"""AdamW over all parameters in a few launches (the reference trains with AdamW:
optimizer/utils.py:8, optimizer/distributed_adamw.py:8), on
``kernels.gradient_norm`` and ``kernels.adamw_step``.
"""
from __future__ import annotations

from itertools import chain
from typing import Callable, Optional, Tuple, Union

import torch
import torch.nn.functional as F

from . import kernels
from .kernels import Moments

_MOMENTS = ("exp_avg", "exp_avg_sq", "scales")


def _refuse_other_updates(group: dict) -> None:
    """Options of torch's groups that name an update which :meth:`AdamW.step` does not make."""
    for name in ("amsgrad", "differentiable"):
        if group.get(name, False):
            raise ValueError(f"{name} is not available: a group with {name}=True would be stepped without it")
    if not group.get("decoupled_weight_decay", True) and group.get("weight_decay", 0.0) != 0.0:
        raise ValueError("a group with decoupled_weight_decay=False (torch.optim.Adam's) would be stepped with decoupled decay")


def _in_8_bits(p: torch.Tensor, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor) -> Moments:
    """fp32 moments of p in 8 bits: the nearest codes, of a root above 0 never that of 0."""
    made, n = kernels.moments(p, 8), p.numel()
    for i, values in enumerate((exp_avg, exp_avg_sq.sqrt())):
        lain = torch.empty_like(p, dtype=torch.float32).copy_(values).as_strided((n,), (1,))  # in the order of memory
        blocks = F.pad(lain, (0, -n % 256)).view(-1, 256)
        top = blocks.abs().amax(1)
        scale = torch.where(top.isfinite(), top / 448, torch.inf)  # infinite: the block is NaN when it is read
        parts = torch.where(scale[:, None] > 0, blocks / scale[:, None], 0.0).clamp(-448.0, 448.0)
        if i == 1:
            parts = torch.where((blocks > 0) & scale.isfinite()[:, None], parts.clamp_min(2.0 ** -9), parts)
        made.scales[i] = scale
        made[i].as_strided((n,), (1,)).copy_(parts.view(-1)[:n])
    return made


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` with fp32 moments whatever the parameters' dtype, or moments in 8
    bits, and with clipping to a norm over all groups in the step itself.

    ``bits``: 32, or 8 for parameters of at least ``min_8bit_size`` elements (see
    :func:`kernels.adamw_step`; smaller ones keep 32).  ``seed`` fixes their random rounding
    (None: from torch's generator, one for all groups that have none of their own; processes that hold replicas of the
    parameters need the same).
    ``max_grad_norm``: gradients are scaled by min(1, max_grad_norm / (norm + 1e-6)) as
    they are read; ``param.grad`` stays as it is, and ``grad_norm`` holds the norm (on
    the device) after a step.  ``skip_nonfinite``: a step whose norm is infinite or
    NaN changes nothing and is not counted.  ``capturable``: the count is kept in device
    memory, so that a step may be captured into a graph (run one before); an
    ``lr`` of a group may then be a one-element fp32 tensor on the device.  See :meth:`replayed`.

    State dicts of ``torch.optim.AdamW`` load (and those of 32-bit moments load there), their moments
    in the bits that the group has; one with
    ``amsgrad`` or ``differentiable``, or of ``torch.optim.Adam`` with a weight decay, raises."""

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, maximize: bool = False, bits: int = 32,
                 min_8bit_size: int = 4096, max_grad_norm: Optional[float] = None, skip_nonfinite: bool = False,
                 capturable: bool = False, seed: Optional[int] = None):
        if bits not in (8, 32):
            raise ValueError(f"moments are held in 32 bits or in 8 (got {bits})")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must be >= 0 (got {lr})")
        if not all(0.0 <= b < 1.0 for b in betas) or len(betas) != 2:
            raise ValueError(f"betas must be two numbers in [0, 1) (got {betas})")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"eps and weight_decay must be >= 0 (got {eps}, {weight_decay})")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"max_grad_norm must be positive (got {max_grad_norm})")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, maximize=maximize,
                                      bits=bits, min_8bit_size=min_8bit_size, seed=None if seed is None else int(seed)))
        self.max_grad_norm, self.skip_nonfinite, self.capturable = max_grad_norm, bool(skip_nonfinite), bool(capturable)
        self.grad_norm: Optional[torch.Tensor] = None
        self._seeds = {}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._seeds = {}

    def __getstate__(self):
        own = {k: v for k, v in self.__dict__.items() if k in ("max_grad_norm", "skip_nonfinite", "capturable", "grad_norm")}
        return {**super().__getstate__(), **own}

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            _refuse_other_updates({**self.defaults, **param_group})
            if param_group.get("bits", self.defaults["bits"]) == 8 and param_group.get("seed") is None:
                param_group["seed"] = self._drawn_seed()
        super().add_param_group(param_group)

    def _drawn_seed(self) -> int:
        """The seed of groups that are given none, drawn when the first of them needs it."""
        if self.defaults["seed"] is None:
            self.defaults["seed"] = int(torch.randint(0, 1 << 62, (1,)).item())
        return self.defaults["seed"]

    def _seed(self, group: dict, device: torch.device) -> torch.Tensor:
        if group["seed"] is None:  # its bits were set later
            group["seed"] = self._drawn_seed()
        seed = group["seed"]
        t = self._seeds.get((seed, device))
        if t is None:
            t = self._seeds[seed, device] = torch.tensor([seed], dtype=torch.int64, device=device)
        return t

    def _begin(self, p: torch.Tensor, group: dict, count) -> dict:
        bits = group["bits"]
        m = kernels.moments(p, 32 if bits == 8 and p.numel() < group["min_8bit_size"] else bits)
        state = self.state[p]
        state["step"] = count
        state.update((k, v) for k, v in zip(_MOMENTS, m) if v is not None)
        return state

    @torch.no_grad()
    def step(self, closure: Optional[Callable] = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        active = [[p for p in group["params"] if p.grad is not None] for group in self.param_groups]
        grads = [p.grad for ps in active for p in ps]
        if not grads:
            return loss
        norm = None
        if self.max_grad_norm is not None or self.skip_nonfinite:
            norm = kernels.gradient_norm(grads, self.max_grad_norm)
            self.grad_norm = norm.norm
        on_device = self.capturable or self.skip_nonfinite
        for index, (group, params) in enumerate(zip(self.param_groups, active)):
            # A tensor's draws go by its place in the group, whichever parameters step together.
            place = {id(p): i for i, p in enumerate(group["params"])} if group["bits"] == 8 else None
            for params, count in self._counted(group, params, on_device, norm):
                moments = [Moments(s["exp_avg"], s["exp_avg_sq"], s.get("scales")) for s in map(self.state.__getitem__, params)]
                kernels.adamw_step(params, [p.grad for p in params], moments, count, lr=group["lr"], betas=group["betas"],
                                   eps=group["eps"], weight_decay=group["weight_decay"], maximize=group["maximize"],
                                   grad_factor=None if norm is None or self.max_grad_norm is None else norm.factor,
                                   found_inf=norm.nonfinite if self.skip_nonfinite else None,
                                   seed=self._seed(group, params[0].device) if group["bits"] == 8 else None,
                                   stream=index, places=None if place is None else [place[id(p)] for p in params])
        return loss

    def replayed(self) -> None:
        """Counts the parameters as changed, which a replay of a captured step does not do by itself: what is derived from
        them outside of the graph and kept until they change (the halves' packed weights in inference) is made anew."""
        params = [p for g in self.param_groups for p in g["params"]]
        torch.autograd.graph.increment_version(p for p in params if not p.is_inference())

    def _counted(self, group, params, on_device, norm):
        """[(parameters, their count with this step)]: those that have taken as many steps, on the host
        by the number, on the device by the counter that they share."""
        sets, made, fresh = {}, {}, None
        for p in params:
            state = self.state[p]
            if "exp_avg" not in state:
                if fresh is None:
                    fresh = torch.zeros(1, dtype=torch.int64, device=p.device) if on_device else 0
                state = self._begin(p, group, fresh)
            count = state["step"]
            if on_device and not isinstance(count, torch.Tensor):  # an option that was set after some steps
                if count not in made:
                    made[count] = torch.tensor([count], dtype=torch.int64, device=p.device)
                count = state["step"] = made[count]
            elif not on_device and isinstance(count, torch.Tensor):
                count = state["step"] = int(count)
            sets.setdefault(id(count) if on_device else count, (count, []))[1].append(p)
        if on_device:  # a parameter that takes no part in this step leaves the others' counter
            left = {}
            taking = set(map(id, params))
            for p in group["params"]:
                count = self.state[p].get("step") if p in self.state and id(p) not in taking else None
                if count is not None and id(count) in sets:
                    left.setdefault(id(count), count.clone())
                    self.state[p]["step"] = left[id(count)]
        out = []
        for count, members in sets.values():
            if on_device:
                count.add_(1 if not self.skip_nonfinite else norm.nonfinite.eq(0))
            else:
                count += 1
                for p in members:
                    self.state[p]["step"] = count
            out.append((members, count))
        return out

    def state_dict(self):
        """As torch's, each parameter with its count as a number (in device memory parameters share a counter, to
        which an optimizer that loads it would add once for each of them)."""
        numbers = {}

        def counted(_, made):  # before the other hooks
            for at, state in made["state"].items():
                count = state.get("step") if isinstance(state, dict) else None
                if isinstance(count, torch.Tensor):
                    if id(count) not in numbers:
                        numbers[id(count)] = int(count)
                    made["state"][at] = {**state, "step": numbers[id(count)]}

        hook = self.register_state_dict_post_hook(counted, prepend=True)
        try:
            return super().state_dict()
        finally:
            hook.remove()

    def load_state_dict(self, state_dict):
        own, given = self.param_groups, []

        def pairs(made):  # its numbers of the parameters, and those
            return zip(*(chain.from_iterable(g["params"] for g in groups) for groups in (made["param_groups"], own)))

        def check(_, made):  # what the hooks before it made of the state dict, before anything is changed
            for group in made["param_groups"]:
                _refuse_other_updates(group)
            for at, p in pairs(made):
                state = made["state"].get(at) or {}
                if state.get("scales") is not None and any(state[k].stride() != p.stride() for k in _MOMENTS[:2]):
                    raise ValueError("moments in 8 bits of a parameter that lay otherwise in memory")
            given.append(made)

        hook = self.register_load_state_dict_pre_hook(check)
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
        state_dict = given[0]
        for group, before in zip(self.param_groups, own):  # torch.optim.AdamW's groups do not have all options
            for name, value in self.defaults.items():
                group.setdefault(name, before.get(name, value))
            if group["seed"] is None:
                group["seed"] = before.get("seed")
            group["betas"] = tuple(group["betas"])
            if "decoupled_weight_decay" in group:
                group["decoupled_weight_decay"] = True
        # Moments keep their own types (the parent casts them to the parameters').
        counters, group_of = {}, {id(p): i for i, g in enumerate(self.param_groups) for p in g["params"]}
        for at, p in pairs(state_dict):
            saved = state_dict["state"].get(at)
            if not saved:
                continue
            state = self.state[p]
            for name in _MOMENTS:
                t = saved.get(name)
                if t is None:
                    continue
                if name == "scales":
                    state[name] = t.detach().to(device=p.device, dtype=torch.float32, copy=True).contiguous()
                    continue
                held = torch.float8_e4m3fn if saved.get("scales") is not None else torch.float32
                state[name] = torch.empty_like(p, dtype=held)
                state[name].copy_(t.to(held))
            group = self.param_groups[group_of[id(p)]]
            if group["bits"] == 8 and "exp_avg" in saved and saved.get("scales") is None and p.numel() >= group["min_8bit_size"]:
                state.update(zip(_MOMENTS, _in_8_bits(p, state["exp_avg"], state["exp_avg_sq"])))
            on_device = self.capturable or self.skip_nonfinite
            count = int(saved["step"])
            if on_device:
                key = (group_of[id(p)], count)
                if key not in counters:
                    counters[key] = torch.tensor([count], dtype=torch.int64, device=p.device)
                count = counters[key]
            state["step"] = count
