"""AdamW over a model's weights in one launch, with moments in 32 or in 8 bits.

The reference's loops construct torch's optimizers (main_imagenet.py:212-213, main_conv.py:232-233); this one takes their
place in ``utils_own.train``: it is a ``torch.optim.Optimizer``, so learning-rate schedulers and ``GradScaler`` work with it
(the latter's scale and its verdict on overflow are applied on the device, without a host synchronisation).
"""
from __future__ import annotations

import copy
from collections import OrderedDict
from collections.abc import Mapping
from typing import Dict

import torch

try:
    from torch.optim.optimizer import _global_optimizer_post_hooks as _POST_HOOKS
    from torch.optim.optimizer import _global_optimizer_pre_hooks as _PRE_HOOKS
except ImportError:  # a torch without hooks for all optimizers
    _PRE_HOOKS, _POST_HOOKS = {}, {}

from . import _lib
from .ops import _DTYPES, _on


class _Views(dict):
    """A parameter's moments: views of the flat buffers.  What is assigned to one of them is copied into it."""

    def __setitem__(self, name, value):
        if name not in self:
            raise KeyError(f"AdamW: a parameter's state has {', '.join(self)}, and no {name}")
        mine, value = self[name], torch.as_tensor(value)
        if value.shape != mine.shape:
            raise ValueError(f"AdamW: expected {name} {tuple(mine.shape)}, got {tuple(value.shape)}")
        if value is not mine:
            with torch.no_grad():
                mine.copy_(value)

    def update(self, *args, **kwargs):
        for name, value in dict(*args, **kwargs).items():
            self[name] = value

    def _refuse(self, *args, **kwargs):
        raise TypeError("AdamW: a parameter's state cannot be taken away; zero_() its tensors")

    __delitem__ = __ior__ = clear = pop = popitem = setdefault = _refuse

    def __reduce__(self):
        # copies and pickles are dictionaries of their own, of a kind that torch.load takes as it is
        return OrderedDict, (), None, None, iter(self.items())


class _State(Mapping):
    """All parameters' views of the flat moment buffers, made when they are asked for.  (It knows the plans and not the
    optimizer: the two would keep one another, and the moments, until a garbage collection.)"""

    def __init__(self, place):
        self._place, self._made = place, {}

    def __getitem__(self, p) -> _Views:
        made = self._made.get(p)
        if made is None:
            made = self._made[p] = _views(*self._place[p])
        return made

    def __setitem__(self, p, value) -> None:
        self[p].update(value)

    def __contains__(self, p) -> bool:
        return p in self._place

    def __iter__(self):
        return iter(self._place)

    def __len__(self) -> int:
        return len(self._place)

    def __reduce__(self):
        return OrderedDict, (), None, None, iter(self.items())


BLOCK = 256  # elements of a block of the flat moment buffers (of a scale of 8-bit moments)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, in fp32 whatever the weights' type:

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps)

    ``params``: dense CUDA tensors in float32, float16 or bfloat16 (others are refused), gradients in any floating-point type.
    ``state_bits=32`` keeps m and v in fp32.  ``state_bits=8`` keeps m and sqrt(v) as e4m3 with an fp32 scale for every 256
    elements, a sixteenth of a byte per weight beside the two: a quarter of the memory.  Their rounding alternates between the
    two neighbouring values so that its mean over the steps is right (rounding to nearest would freeze them); it depends on the
    element's place and the step count alone, so runs repeat.  A gradient that is no finite number spoils its element, with 8
    bits its block of 256.

    ``state`` holds every parameter from the start on; its tensors are views of the buffers (:meth:`flat_state`), and what is
    assigned to them is copied.  An optimizer cannot be copied or pickled: use :meth:`state_dict`.

    A step counts as a write of every weight that has a gradient, also where ``found_inf``, which only the device knows, cancels
    it: a graph that still needs the weights of before raises.

    ``lr`` may be a one-element float32 CUDA tensor, which a captured step then reads at every replay.  The number of steps
    is kept on the device, one count for each parameter group: weights without a gradient are left out of a step, but share
    their group's count.  16-bit weights are rounded to nearest at every step; there is no 32-bit copy of them."""

    _step_supports_amp_scaling = True  # GradScaler hands over grad_scale / found_inf instead of unscaling by itself

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32 (got {state_bits})")
        self._state_bits = state_bits
        self._plans = []
        self._place = {}    # parameter -> (its group's plan, its number there)
        self._built = False
        self._state = _State(self._place)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._built = True

    @property
    def state(self) -> _State:
        return self._state

    @state.setter
    def state(self, value) -> None:
        if self._built:  # (the base class begins with an empty one)
            raise TypeError("AdamW: the state cannot be replaced: use load_state_dict(), or assign to its tensors")

    def __getstate__(self):
        raise TypeError("rexsc_b200.optim.AdamW cannot be copied or pickled: use state_dict()")

    # -- construction -------------------------------------------------------------------------------------------
    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        params = self.param_groups[-1]["params"]
        try:
            if len(set(params)) != len(params):
                raise ValueError("AdamW: a parameter appears twice in its group")
            self._check_apart()
            plan = self._plan(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise
        self._plans.append(plan)
        self._place.update((p, (plan, i)) for i, p in enumerate(params))

    def _plan(self, group) -> dict:
        """Flat moment buffers of a group, every tensor on a block of its own."""
        self._check_numbers(group)
        params = group["params"]
        if not params:
            raise ValueError("AdamW: a parameter group without parameters")
        dev = params[0].device
        for p in params:
            if not p.is_cuda or p.device != dev:
                raise ValueError("AdamW: the parameters of a group must be on one CUDA device")
            if p.dtype not in _DTYPES:
                raise ValueError(f"AdamW: parameters must be float32, float16 or bfloat16 (got {p.dtype})")
            if not _dense(p) or p.is_neg():
                raise ValueError("AdamW: parameters must be dense (no gaps or overlaps between their elements)")
        sizes = [p.numel() for p in params]
        blocks = [-(-n // BLOCK) for n in sizes]
        first = [0]
        for b in blocks:
            first.append(first[-1] + b)
        total = first[-1] * BLOCK
        with _on(dev):
            zeros = lambda n, t: torch.zeros(n, dtype=t, device=dev)
            if self._state_bits == 32:
                flat = {"exp_avg": zeros(total, torch.float32), "exp_avg_sq": zeros(total, torch.float32)}
            else:
                flat = {"exp_avg": zeros(total, torch.uint8).view(torch.float8_e4m3fn),
                        "exp_avg_sqrt": zeros(total, torch.uint8).view(torch.float8_e4m3fn),
                        "exp_avg_scale": zeros(first[-1], torch.float32),
                        "exp_avg_sqrt_scale": zeros(first[-1], torch.float32)}
            step = zeros(2, torch.int64)
        second = "exp_avg_sq" if self._state_bits == 32 else "exp_avg_sqrt"
        native = _lib.host().AdamWPlan(params, self._state_bits, step, flat["exp_avg"], flat[second], flat.get("exp_avg_scale"),
                                       flat.get("exp_avg_sqrt_scale"))
        return {"flat": flat, "step": step, "native": native, "first": first, "shapes": [p.shape for p in params],
                "strides": [p.stride() for p in params]}

    def _check_apart(self) -> None:
        """One launch updates all tensors at once: no two of them may hold the same element."""
        spans = sorted((p.device.index or 0, p.data_ptr(), p.data_ptr() + p.numel() * p.element_size())
                       for g in self.param_groups for p in g["params"] if p.is_cuda and p.numel())
        for (dev, _, end), (next_dev, begin, _) in zip(spans, spans[1:]):
            if dev == next_dev and begin < end:
                raise ValueError("AdamW: two parameters share memory")

    @staticmethod
    def _check_numbers(group) -> None:
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1:
                raise ValueError("AdamW: lr must have one element")
        elif not lr >= 0:
            raise ValueError(f"AdamW: lr must not be negative (got {lr})")
        if not (0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError(f"AdamW: betas must lie in [0, 1) (got {b1}, {b2})")
        if not (group["eps"] >= 0 and group["weight_decay"] >= 0):
            raise ValueError("AdamW: eps and weight_decay must not be negative")
        if group["eps"] and not 2.0 ** -126 <= group["eps"] < 2.0 ** 126:
            raise ValueError(f"AdamW: eps must be 0 or a normal number in fp32 (got {group['eps']})")

    def flat_state(self, group: int = 0) -> Dict[str, torch.Tensor]:
        """The buffers that hold the moments of a parameter group, and its step count: ``exp_avg`` and ``exp_avg_sq`` (fp32),
        or ``exp_avg`` and ``exp_avg_sqrt`` (e4m3) with their ``*_scale``.  Tensor i of the group begins on the first block
        of 256 elements behind tensor i - 1, in the order of its memory.  Writing to them changes the optimizer's state."""
        plan = self._plans[group]
        return {**plan["flat"], "step": plan["step"][0]}

    # -- checkpoints --------------------------------------------------------------------------------------------
    def state_dict(self):
        """As torch's optimizers give it; the tensors are the optimizer's own.  Moments in 8 bits are stored in the order of
        the weights' memory."""
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        number = {p: i for i, p in enumerate(self.state)}
        groups = [{**group, "params": [number[p] for p in group["params"]], "strides": [tuple(s) for s in plan["strides"]]}
                  for group, plan in zip(self.param_groups, self._plans)]
        sd = {"state": {number[p]: dict(views) for p, views in self.state.items()}, "param_groups": groups,
              "state_bits": self._state_bits}
        for hook in self._optimizer_state_dict_post_hooks.values():
            changed = hook(self, sd)
            if changed is not None:
                sd = changed
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """Takes over copies of a state's moments and numbers, none of its tensors.  Where a group's ``lr`` is a tensor it stays
        that tensor and gets the saved value, so that a captured step goes on reading the right one."""
        state_dict = state_dict.copy()
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            if changed is not None:
                state_dict = changed
        groups = state_dict["param_groups"]
        if state_dict.get("state_bits") != self._state_bits:
            raise ValueError(f"AdamW: the state was saved with state_bits={state_dict.get('state_bits')}, not {self._state_bits}")
        if len(groups) != len(self.param_groups) or any(len(a["params"]) != len(b["params"])
                                                        for a, b in zip(groups, self.param_groups)):
            raise ValueError("AdamW: the state has other parameter groups")
        todo = []
        for group, saved, plan in zip(self.param_groups, groups, self._plans):
            self._check_numbers(saved)
            strides = saved["strides"]
            for i, (p, key) in enumerate(zip(group["params"], saved["params"])):
                if self._state_bits == 8 and tuple(strides[i]) != tuple(plan["strides"][i]):
                    raise ValueError("AdamW: 8-bit moments of a weight with another memory format cannot be loaded")
                mine, theirs = self.state[p], state_dict["state"][key]
                if set(mine) != set(theirs) or any(mine[n].shape != theirs[n].shape for n in mine):
                    raise ValueError("AdamW: the state has moments of another shape")
                todo += [(mine[n], theirs[n]) for n in mine]
        for mine, theirs in todo:
            mine.copy_(theirs)
        for group, saved in zip(self.param_groups, groups):
            lr = group["lr"]
            group.update({k: copy.deepcopy(v) for k, v in saved.items() if k not in ("params", "param_names", "strides")})
            if isinstance(lr, torch.Tensor):
                lr.copy_(torch.as_tensor(group["lr"]).reshape(lr.shape))
                group["lr"] = lr
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    # -- step ---------------------------------------------------------------------------------------------------
    def step(self, closure=None):
        args, kwargs = (self,) if closure is None else (self, closure), {}
        for hook in (*_PRE_HOOKS.values(), *self._optimizer_step_pre_hooks.values()):
            changed = hook(self, args, kwargs)
            if changed is not None:
                if not isinstance(changed, tuple) or len(changed) != 2:
                    raise RuntimeError(f"AdamW: a step's pre-hook must return None or (args, kwargs), not {changed}")
                args, kwargs = changed
                closure = _closure_of(*args, **kwargs)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        scale, inf = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        for group, plan in zip(self.param_groups, self._plans):
            lr, (b1, b2) = group["lr"], group["betas"]
            on_device = isinstance(lr, torch.Tensor) and lr.is_cuda
            plan["native"].step(group["params"], 0.0 if on_device else float(lr), lr if on_device else None, b1, b2,
                                group["eps"], group["weight_decay"], scale, inf)
        for hook in (*self._optimizer_step_post_hooks.values(), *_POST_HOOKS.values()):
            hook(self, args, kwargs)
        return loss

    # torch wraps an optimizer's step in a profiler range and calls the hooks there, 10 us of the host's time in a step
    # whose launch takes 4; the hooks are called above instead
    step.hooked = True


def _views(plan: dict, i: int) -> _Views:
    """Of parameter i of a group's plan."""
    first, last, shape, stride = plan["first"][i], plan["first"][i + 1], plan["shapes"][i], plan["strides"][i]
    views = {"step": plan["step"][0]}
    for name, t in plan["flat"].items():
        if name.endswith("_scale"):
            views[name] = t[first:last]
        else:
            views[name] = t.as_strided(shape, stride, first * BLOCK) if last > first else t[:0].view(shape)
    return _Views(views)


def _closure_of(optimizer, closure=None):
    """The closure among a step's arguments as a hook has left them."""
    return closure


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements of a tensor fill a contiguous piece of memory, each its own place."""
    expected = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda x: x[1]):
        if stride != expected:
            return False
        expected *= size
    return True
