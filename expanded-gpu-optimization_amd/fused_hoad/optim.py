"""AdamW for networks of many tensors, with moments in 32 or in 8 bits, as HIP kernels."""

from __future__ import annotations

import math
from collections.abc import Callable, Iterable
from itertools import chain
from operator import is_

import torch
from torch import Tensor

from fused_hoad._extension import adamw_step, load_extension

#: Values of packed state that share a scale; every tensor's state starts at a multiple of it.
STATE_BLOCK = 256


def state_span(numel: int) -> int:
    """Values that a tensor of ``numel`` elements takes in a packed state."""
    return -(-numel // STATE_BLOCK) * STATE_BLOCK


def packed_state_size(parameters: Iterable[Tensor]) -> int:
    """Values of a packed state of these tensors."""
    return sum(state_span(p.numel()) for p in parameters)


def _check_options(group: dict) -> None:
    """Raises ``ValueError`` for options that a step does not take or would not heed."""
    if not group["lr"] >= 0.0 or not group["eps"] >= 0.0 or not group["weight_decay"] >= 0.0:
        raise ValueError("lr, eps and weight_decay must be non-negative")
    beta1, beta2 = group["betas"]
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError("betas must lie in [0, 1)")
    if group["state_bits"] not in (8, 32):
        raise ValueError("state_bits must be 8 or 32")
    if not 0 <= group["seed"] < 2**32:
        raise ValueError("seed must fit 32 bits")
    if group.get("amsgrad") or group.get("maximize"):
        raise ValueError("amsgrad and maximize are not supported")
    if group["weight_decay"] and not group.get("decoupled_weight_decay", True):
        raise ValueError("weight_decay that is not decoupled is not supported")


class FusedAdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` (decoupled weight decay; no amsgrad, no maximize) as one native call
    a parameter group: two kernels for every 108 tensors, whatever their sizes.

    ``state_bits=32`` keeps both moments in float32; ``state_bits=8`` keeps a byte for each, the
    first moment and the second moment's square root as small floating-point numbers over a scale
    that 256 values share, a quarter of the memory. They are rounded stochastically, so that the slow
    second moment keeps moving (its relative change per step is far below a code's spacing), by bits
    mixed from ``seed``, the step and the place: runs are reproducible.

    Parameters are contiguous float32 or bfloat16 CUDA tensors, one device to a group; the update is
    formed in float32 and rounded once. A parameter without a gradient is left alone and its step
    not counted. The step counts live on the device and nothing synchronises, so a step can be
    captured in a HIP graph (after a first step, which allocates the state; the options of the group
    are then those of the capture). ``load_state_dict`` writes into the state that is there, and a captured
    step goes on from what was loaded; only with other ``state_bits`` or on another device the state is a new
    one, and a step has to be captured again.

    The moments of a group are packed in a few tensors; ``state[p]`` holds views of them
    (``exp_avg`` and ``exp_avg_sq`` in ``p``'s shape, or in 8 bits the blocks' codes and their
    ``exp_avg_scale`` and ``exp_avg_sq_scale``; ``step``, int32), so ``state_dict`` and
    ``load_state_dict`` work as usual. What ``state`` and the groups hold counts: entries that were taken out
    start again from zero, and tensors that were put in place of the views are copied in.
    """

    def __init__(
        self,
        params,
        lr: float = 1e-3,
        betas: tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 1e-2,
        *,
        state_bits: int = 32,
        seed: int = 0,
    ) -> None:
        super().__init__(
            params,
            {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay,
             "state_bits": state_bits, "seed": seed},
        )

        self._packs: dict[int, dict[str, Tensor | None]] = {}
        self._members: dict[int, list[Tensor]] = {}  # the parameters of each
        self._seen: list[Tensor] = []

    def add_param_group(self, param_group: dict) -> None:
        """Adds a group, with the defaults for options that it does not give."""
        _check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        self._packs, self._members, self._seen = {}, {}, []  # made again from self.state

    def _tensors(self) -> list[Tensor]:
        """The groups' parameters and what ``self.state`` holds."""
        return [*chain.from_iterable(group["params"] for group in self.param_groups),
                *chain.from_iterable(map(dict.values, self.state.values()))]

    def _update_packs(self) -> None:
        """Packs the groups' state where it is not the one of the last step: a first step, a new group, a
        copied optimizer, parameters or state that were changed from outside. Values come from ``self.state``;
        the packed state of the same parameters is kept."""
        if load_extension().same_objects([group["params"] for group in self.param_groups], self.state, self._seen):
            return
        for index, group in enumerate(self.param_groups):
            if not group["params"]:
                continue
            packed, views = self._present(index, group) or self._pack(group)
            self._fill(group, views, {p: {name: value for name, value in self.state[p].items() if name in views[p]}
                                      for p in group["params"]})
            self._packs[index], self._members[index] = packed, list(group["params"])
            for p, own in views.items():
                self.state[p].update(own)
        self._seen = self._tensors()

    def _present(self, index: int, group: dict):
        """Group ``index``'s packed state and its views, if it is of these parameters, on their device and has
        the moments' width that ``group`` asks for; else ``None``."""
        packed, params = self._packs.get(index), group["params"]
        if packed is None or len(params) != len(self._members[index]) or not all(map(is_, params, self._members[index])):
            return None
        moment = packed["exp_avg"]
        if (moment.dtype == torch.uint8) != (group["state_bits"] == 8) or any(p.device != moment.device for p in params):
            return None
        return packed, self._views(params, packed)

    @staticmethod
    def _pack(group: dict) -> tuple[dict[str, Tensor | None], dict[Tensor, dict[str, Tensor]]]:
        """A packed state of zeros for the group, and its views by parameter."""
        params, eight = group["params"], group["state_bits"] == 8
        device = params[0].device
        if any(p.device != device for p in params):
            raise ValueError("a parameter group must be on one device")
        size = packed_state_size(params)
        dtype = torch.uint8 if eight else torch.float32
        packed: dict[str, Tensor | None] = {
            "exp_avg": torch.zeros(size, dtype=dtype, device=device),
            "exp_avg_sq": torch.zeros(size, dtype=dtype, device=device),
            "step": torch.zeros(len(params), dtype=torch.int32, device=device),
            "exp_avg_scale": torch.zeros(size // STATE_BLOCK, device=device) if eight else None,
            "exp_avg_sq_scale": torch.zeros(size // STATE_BLOCK, device=device) if eight else None,
        }
        return packed, FusedAdamW._views(params, packed)

    @staticmethod
    def _views(params: list[Tensor], packed: dict[str, Tensor | None]) -> dict[Tensor, dict[str, Tensor]]:
        """What of a packed state belongs to each parameter."""
        eight = packed["exp_avg_scale"] is not None
        every: dict[Tensor, dict[str, Tensor]] = {}
        at = 0
        for k, p in enumerate(params):
            span = state_span(p.numel())
            views = every[p] = {"step": packed["step"][k]}
            for name in ("exp_avg", "exp_avg_sq"):
                values = packed[name][at : at + span]
                views[name] = values if eight else values[: p.numel()].view(p.shape)
                if eight:
                    scales = packed[name + "_scale"]
                    views[name + "_scale"] = scales[at // STATE_BLOCK : (at + span) // STATE_BLOCK]
            at += span
        return every

    @staticmethod
    def _check(group: dict, every: dict[Tensor, dict[str, Tensor]], states) -> None:
        """Raises unless each parameter's views take what ``states`` has for it."""
        for p, views in every.items():
            for name, value in states.get(p, {}).items():
                if name not in views or views[name].shape != value.shape or (
                    name != "step" and views[name].dtype != value.dtype
                ):
                    raise ValueError(f"state {name!r} does not fit a parameter of shape {tuple(p.shape)} "
                                     f"with {group['state_bits']}-bit moments")

    @classmethod
    @torch.no_grad()
    def _fill(cls, group: dict, every: dict[Tensor, dict[str, Tensor]], states) -> None:
        """Writes into each parameter's views what ``states`` has for it, and zeros what it has not."""
        cls._check(group, every, states)
        for p, views in every.items():
            given = states.get(p, {})
            for name, view in views.items():
                value = given.get(name)
                if value is None:
                    view.zero_()
                elif value.data_ptr() != view.data_ptr() or value.dtype != view.dtype:  # not this memory itself
                    view.copy_(value)

    @torch.no_grad()
    def step(self, closure: Callable[[], Tensor] | None = None) -> Tensor | None:
        """One step; ``closure``, if given, is evaluated first and its value returned."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._update_packs()
        for index, group in enumerate(self.param_groups):
            if not group["params"]:
                continue
            packed = self._packs[index]
            adamw_step(
                group["params"],
                [p.grad for p in group["params"]],
                packed["exp_avg"],
                packed["exp_avg_sq"],
                packed["step"],
                lr=group["lr"],
                betas=group["betas"],
                eps=group["eps"],
                weight_decay=group["weight_decay"],
                exp_avg_scale=packed["exp_avg_scale"],
                exp_avg_sq_scale=packed["exp_avg_sq_scale"],
                seed=group["seed"],
            )
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """Options and state of ``state_dict``, whose groups must match this optimizer's. The values
        are copied into the packed state with their own types (the base class would cast the moments to
        the parameters' type): into the present one where it has the same layout, else into a new one.
        Nothing is changed when something does not fit."""
        state_dict = dict(state_dict)  # a hook may change it
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            given = hook(self, state_dict)
            state_dict = state_dict if given is None else given
        saved = state_dict["param_groups"]
        if [len(g["params"]) for g in saved] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the state's parameter groups do not match the optimizer's")
        merged, packs, fills = [], {}, []
        for index, (group, other) in enumerate(zip(self.param_groups, saved, strict=True)):
            merged.append({**group, **other, "params": group["params"]})
            _check_options(merged[-1])
            if not group["params"]:
                continue
            states = {p: state_dict["state"].get(key, {})
                      for p, key in zip(group["params"], other["params"], strict=True)}
            packs[index], views = self._present(index, merged[-1]) or self._pack(merged[-1])
            self._check(merged[-1], views, states)
            fills.append((merged[-1], views, states))
        for fill in fills:
            self._fill(*fill)
        for group, options in zip(self.param_groups, merged, strict=True):
            group.update(options)
        self._packs = packs
        self._members = {index: list(self.param_groups[index]["params"]) for index in packs}
        self.state.clear()
        for _, views, _ in fills:
            self.state.update(views)
        self._seen = self._tensors()
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def moments(self, parameter: Tensor) -> tuple[Tensor, Tensor]:
        """``parameter``'s first and second moments in float32 and its shape."""
        from fused_hoad._extension import decode_moments

        state = self.state[parameter]
        if "exp_avg_scale" not in state:
            return state["exp_avg"].clone(), state["exp_avg_sq"].clone()
        mean, square = decode_moments(*(state[name] for name in
                                        ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")))
        numel = math.prod(parameter.shape)
        return mean[:numel].view(parameter.shape), square[:numel].view(parameter.shape)
