"""AdamW over a model's weights in one launch, with moments in 32 or in 8 bits.

The reference's loops construct torch's optimizers (main_imagenet.py:212-213, main_conv.py:232-233); this one takes their
place in ``utils_own.train``: it is a ``torch.optim.Optimizer``, so learning-rate schedulers and ``GradScaler`` work with it
(the latter's scale and its verdict on overflow are applied on the device, without a host synchronisation).
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import Dict

import numpy as np
import torch

try:
    from torch.optim.optimizer import _global_optimizer_post_hooks as _POST_HOOKS
    from torch.optim.optimizer import _global_optimizer_pre_hooks as _PRE_HOOKS
except ImportError:  # a torch without hooks for all optimizers
    _PRE_HOOKS, _POST_HOOKS = {}, {}

from . import _lib
from .ops import _DTYPES, _on, _stream

_STRIDED = torch.strided
_stride, _numel, _data_ptr, _dtype = (torch.Tensor.stride, torch.Tensor.numel, torch.Tensor.data_ptr,
                                      operator.attrgetter("dtype"))
BLOCK = 256  # elements of a block of the flat moment buffers (of a scale of 8-bit moments)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, in fp32 whatever the weights' type:

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps)

    ``params``: dense CUDA tensors in float32, float16 or bfloat16, gradients in any of these.  ``state_bits=32`` keeps m and
    v in fp32.  ``state_bits=8`` keeps m and sqrt(v) as e4m3 with an fp32 scale for every 256 elements, a sixteenth of a byte
    per weight beside the two: a quarter of the memory.  Their rounding alternates between the two neighbouring values so that
    its mean over the steps is right (rounding to nearest would freeze them); it depends on the element's place and the step
    count alone, so runs repeat.  A gradient that is no finite number spoils its element, with 8 bits its block of 256.

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
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        raise TypeError("rexsc_b200.optim.AdamW cannot be copied or pickled: use state_dict()")

    # -- construction -------------------------------------------------------------------------------------------
    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        try:
            self._plans.append(self._plan(self.param_groups[-1]))
        except Exception:
            self.param_groups.pop()
            raise

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
            if not _dense(p):
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
        table = np.zeros((len(params), 4), dtype=np.int64)  # rexsc_adamw_tensor: param, grad, numel, first_block
        table[:, 2], table[:, 3] = sizes, first[:-1]
        for i, p in enumerate(params):
            a, b = first[i] * BLOCK, first[i] * BLOCK + sizes[i]
            views = {}
            for name, t in flat.items():
                if name.endswith("_scale"):
                    views[name] = t[first[i]:first[i + 1]]
                else:
                    views[name] = t[a:b].as_strided(p.shape, p.stride()) if b > a else t[a:b].view(p.shape)
            self.state[p] = {"step": step[0], **views}
        d = _lib.AdamWDesc()
        d.state_bits = self._state_bits
        second = "exp_avg_sq" if self._state_bits == 32 else "exp_avg_sqrt"
        d.d_step, d.d_exp_avg, d.d_exp_avg_sq = step.data_ptr(), flat["exp_avg"].data_ptr(), flat[second].data_ptr()
        if self._state_bits == 8:
            d.d_exp_avg_scale = flat["exp_avg_scale"].data_ptr()
            d.d_exp_avg_sq_scale = flat["exp_avg_sqrt_scale"].data_ptr()
        return {"flat": flat, "step": step, "table": table, "desc": d, "device": dev, "sizes": sizes,
                "strides": [p.stride() for p in params]}

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
        sd = super().state_dict()
        sd["state_bits"] = self._state_bits
        for i, (strides, plan) in enumerate((p["strides"], p) for p in self._plans):
            sd["param_groups"][i]["strides"] = [tuple(s) for s in strides]
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
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
            group.update({k: v for k, v in saved.items() if k not in ("params", "strides")})

    # -- step ---------------------------------------------------------------------------------------------------
    def step(self, closure=None):
        for hook in (*_PRE_HOOKS.values(), *self._optimizer_step_pre_hooks.values()):
            changed = hook(self, (self, closure), {})
            if changed is not None:
                closure = changed[0][1]
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group, plan in zip(self.param_groups, self._plans):
            self._step_group(group, plan)
        for hook in (*self._optimizer_step_post_hooks.values(), *_POST_HOOKS.values()):
            hook(self, (self, closure), {})
        return loss

    # torch wraps an optimizer's step in a profiler range and calls the hooks there, 10 us of the host's time in a step
    # whose launch takes 4; the hooks are called above instead
    step.hooked = True

    def _gather(self, group, plan):
        """Parameters that take part in a step, their gradients in the parameters' order of memory, and their places."""
        params, strides, sizes = group["params"], plan["strides"], plan["sizes"]
        grads = [p.grad for p in params]
        # whole lists at a time: a loop over the tensors costs the host twice as much
        try:
            ordinary = (list(map(_stride, grads)) == strides and list(map(_numel, grads)) == sizes
                        and list(map(_stride, params)) == strides and list(map(_numel, params)) == sizes and 0 not in sizes)
        except (TypeError, RuntimeError):   # a gradient that is None, or has no strides (sparse)
            ordinary = False
        if ordinary:
            return params, grads, plan["table"].copy()
        chosen, kept = [], []
        for i, (p, g) in enumerate(zip(params, grads)):
            if g is None or sizes[i] == 0:
                continue
            if p.stride() != strides[i] or p.numel() != sizes[i] or p.device != plan["device"]:
                raise ValueError("AdamW: a parameter has changed its size, memory format or device")
            if g.layout is not _STRIDED:
                raise ValueError("AdamW: sparse gradients are not supported")
            if g.stride() != strides[i] or g.numel() != sizes[i]:
                g = torch.empty_strided(p.shape, strides[i], dtype=g.dtype, device=g.device).copy_(g.detach())
            chosen.append(i)
            kept.append(g)
        return [params[i] for i in chosen], kept, plan["table"][chosen]

    def _step_group(self, group, plan) -> None:
        params, grads, table = self._gather(group, plan)
        if not params:
            return
        kinds = list(zip(map(_dtype, params), map(_dtype, grads)))
        distinct = set(kinds)
        for pair in distinct:
            if pair[0] not in _DTYPES:
                raise ValueError(f"AdamW: parameters must be float32, float16 or bfloat16 (got {pair[0]})")
        if any(pair[1] not in _DTYPES for pair in distinct):
            grads = [g if g.dtype in _DTYPES else g.detach().float() for g in grads]
            kinds = list(zip(map(_dtype, params), map(_dtype, grads)))
            distinct = set(kinds)
        table[:, 0] = list(map(_data_ptr, params))
        table[:, 1] = list(map(_data_ptr, grads))
        dev, flat, d = plan["device"], plan["flat"], plan["desc"]
        d.beta1, d.beta2 = group["betas"]
        d.eps, d.weight_decay = group["eps"], group["weight_decay"]
        keep = []
        lr = group["lr"]
        if isinstance(lr, torch.Tensor) and lr.is_cuda:
            keep.append(lr.detach().to(device=dev, dtype=torch.float32))
            d.d_lr, d.lr = keep[-1].data_ptr(), 0.0
        else:
            d.d_lr, d.lr = None, float(lr)
        d.d_grad_scale = d.d_found_inf = None
        for name in ("grad_scale", "found_inf"):
            t = getattr(self, name, None)
            if t is not None:
                if t.device != dev or t.dtype is not torch.float32:
                    t = t.to(device=dev, dtype=torch.float32)
                keep.append(t)
                setattr(d, "d_" + name, t.data_ptr())
        launch = _lib.load().rexsc_adamw_step
        with _on(dev):
            stream = _stream(dev)
            for j, kind in enumerate(distinct):
                part = table if len(distinct) == 1 else np.ascontiguousarray(table[[k == kind for k in kinds]])
                d.param_dtype, d.grad_dtype = _DTYPES[kind[0]], _DTYPES[kind[1]]
                d.advance = j == len(distinct) - 1
                rc = launch(C.byref(d), part.ctypes.data, len(part), stream)
                if rc:
                    _lib.check(rc, "rexsc_adamw_step")


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements of a tensor fill a contiguous piece of memory, each its own place."""
    expected = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda x: x[1]):
        if stride != expected:
            return False
        expected *= size
    return True
