"""AdamW on torch CUDA tensors: one call updates every tensor of a model.

* ``AdamW``, a ``torch.optim.Optimizer``: 16-bit parameters keep a float32 master, the
  moments are float32 or 8 bits (``moment_bits=8``);
* ``adamw_step``, the step by itself on lists of tensors, and ``moment_values``, what the
  codes of an 8-bit moment stand for.

The calls are the entry points so3lr_adamw and so3lr_moment_values of
include/so3lr_b200.h, which has the formulas, through the compiled module of the
feed-forward layers; its conventions hold here: kernels are queued on the current torch
stream of the tensors' GPU, arguments that do not fit one another raise ValueError, a
value outside the library's range So3lrError, and there is no CPU path. The step
counters are on the GPU, so a step may be captured in a graph and replayed.
"""
from __future__ import annotations

import torch

from .layers import _layers

__all__ = ["AdamW", "adamw_step", "moment_values", "SCALE_BLOCK"]

SCALE_BLOCK = 256  # elements of a tensor that share the scale of an 8-bit moment


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, exp_avg_scales=None, exp_avg_sq_scales=None,
               masters=None, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2) -> None:
    """One AdamW step of lists of contiguous tensors, in place:

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

    params: float32, bfloat16 or float16; grads: the parameter's type or float32. steps: the
    counters t, to which the call adds 1: an int64 tensor of one element for each parameter,
    or a list of one-element tensors. masters: for each parameter a float32 tensor that is
    updated in its place, the parameter being its rounding, or None. Moments are float32; with
    a tensor of scales for a parameter, one for each 256 elements, 8 bits (exp_avgs int8,
    exp_avg_sqs uint8). lr: a number, or a float32 tensor of one element on the GPU, which is
    read there. Zero codes and scales are zero moments. Nothing in the call may overlap;
    parameters or counters that do are refused."""
    _layers.adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, exp_avg_scales, exp_avg_sq_scales, masters, lr,
                       *betas, eps, weight_decay)


def moment_values(codes, scales, dtype=torch.float32):
    """What an 8-bit moment's codes stand for, rounded to dtype: scales[i / 256] c |c| / 127^2
    for int8 codes (the first moment), scales[i / 256] (c / 255)^4 for uint8 (the second)."""
    return _layers.moment_values(codes, scales, dtype)


def _copied(p, copies):
    """A contiguous copy of a parameter of another layout, noted in copies."""
    reach = 1  # of the dimensions so far, from the shortest stride on
    for stride, size in sorted((t, n) for t, n in zip(p.stride(), p.shape) if n > 1):
        if stride < reach:
            raise ValueError(f"params: elements of a parameter share memory (shape {tuple(p.shape)}, strides {p.stride()})")
        reach = stride * size
    copy = p.contiguous()
    copies.append((p, copy))
    return copy


def _share_memory(a, b):
    """Whether tensors share memory: whether k_i elements of each stride, as many as they have, make up the distance
    between them."""
    sizes = {}  # stride in bytes -> how far a and b go along it
    for side, t in enumerate((a, b)):
        for stride, n in ((1, t.element_size()), *((s * t.element_size(), n) for s, n in zip(t.stride(), t.shape))):
            if n > 1:
                sizes.setdefault(stride, [0, 0])[side] += n - 1
    strides = sorted(sizes, reverse=True)
    reach = [[sum(s * sizes[s][side] for s in strides[i:]) for side in (0, 1)] for i in range(len(strides) + 1)]

    def found(i, distance):
        if i == len(strides):
            return distance == 0
        s, (up, down) = strides[i], sizes[strides[i]]
        least, most = max(-down, -((reach[i + 1][0] - distance) // s)), min(up, (distance + reach[i + 1][1]) // s)
        return any(found(i + 1, distance - k * s) for k in range(least, most + 1))

    return found(0, b.data_ptr() - a.data_ptr())


def _check_apart(params):
    """Refuses parameters that share memory where one is updated in a copy: it would be written over the other's step."""
    size = lambda p: (1 + sum((n - 1) * s for n, s in zip(p.shape, p.stride()))) * p.element_size()  # noqa: E731
    before = []  # those whose memory may reach the next one's
    for p in sorted((p for p in params if p.numel()), key=lambda p: p.data_ptr()):
        before = [q for q in before if q.data_ptr() + size(q) > p.data_ptr()]
        for q in before:
            if not (p.is_contiguous() and q.is_contiguous()) and _share_memory(q, p):
                raise ValueError(f"params: parameters of shapes {tuple(q.shape)} and {tuple(p.shape)} share memory")
        before.append(p)


class AdamW(torch.optim.Optimizer):
    """AdamW over all parameters of a group in one call.

    moment_bits: 32, or 8 (a quarter of the memory; tensors of fewer than 4096 elements keep
    32). master: keep a float32 copy of each 16-bit parameter, made at its first step, and
    update that; the parameter is its rounding, so what is written into a parameter after
    that step is lost. Each may be set for a group. lr may be a float32 tensor of one
    element on the GPU, for graphs. The first step allocates the state: take it before a
    capture. Parameters of a layout that is not contiguous are updated in a contiguous copy
    and written back, which costs a copy each way; their state is contiguous. A group may span
    several GPUs (with a rate that is a number)."""

    SMALL = 4096

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 moment_bits: int = 32, master: bool = True):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, moment_bits=moment_bits,
                                      master=master))

    def add_param_group(self, param_group):
        bits = param_group.get("moment_bits", self.defaults["moment_bits"])
        if bits not in (8, 32):
            raise ValueError(f"moment_bits must be 8 or 32, got {bits}")
        super().add_param_group(param_group)

    def _start(self, p, group):
        state = self.state[p]
        state["step"] = torch.zeros((), dtype=torch.int64, device=p.device)
        flat = dict(device=p.device, memory_format=torch.contiguous_format)
        if group["moment_bits"] == 8 and p.numel() >= self.SMALL:
            blocks = (p.numel() + SCALE_BLOCK - 1) // SCALE_BLOCK
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.int8, **flat)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8, **flat)
            state["exp_avg_scale"], state["exp_avg_sq_scale"] = (torch.zeros(blocks, device=p.device) for _ in range(2))
        else:
            state["exp_avg"], state["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.float32, **flat) for _ in range(2))
        if group["master"] and p.dtype != torch.float32:
            state["master"] = p.detach().float().clone(memory_format=torch.contiguous_format)
        return state

    def _call(self, group, params, fresh):
        """The arguments of the group's adamw_step; parameters whose state is made for it are added to fresh."""
        grads = [g if g.is_sparse or g.is_contiguous() else g.contiguous() for g in [p.grad for p in params]]
        states = [self.state[p] or fresh.append(p) or self._start(p, group) for p in params]
        pick = lambda key: [s.get(key) for s in states]  # noqa: E731
        return (params, grads, pick("exp_avg"), pick("exp_avg_sq"), pick("step"), pick("exp_avg_scale"),
                pick("exp_avg_sq_scale"), pick("master"), group["lr"], *group["betas"], group["eps"], group["weight_decay"])

    @torch.no_grad()
    def step(self, closure=None):
        """One step of every group, or none: what a group's call would refuse is refused before any is queued."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls, fresh, copies = [], [], []
        try:
            for group in self.param_groups:
                params = [p for p in group["params"] if p.grad is not None]
                if _layers.uniform(params):
                    calls += [self._call(group, params, fresh)] if params else []
                else:
                    for device in sorted({p.device for p in params}, key=str):
                        there = [p for p in params if p.device == device]
                        call = self._call(group, there, fresh)
                        calls.append(([p if p.is_contiguous() else _copied(p, copies) for p in there], *call[1:]))
            if copies:
                _check_apart([p for group in self.param_groups for p in group["params"] if p.grad is not None])
            _layers.adamw_steps(calls)
        except Exception:
            for p in fresh:  # a master made now would be stale if the weights change before the next step
                self.state.pop(p, None)
            raise
        for p, updated in copies:
            p.copy_(updated)
        return loss

    def load_state_dict(self, state_dict):
        """As torch.optim.Optimizer's, with each state tensor in its own type: the base class
        would cast masters, moments and scales to the parameter's."""
        loaded = {}

        def restore(optimizer):
            saved = [i for g in loaded["param_groups"] for i in g["params"]]
            params = [p for g in optimizer.param_groups for p in g["params"]]
            for i, p in zip(saved, params):
                if i in loaded["state"]:
                    optimizer.state[p] = {k: v.to(p.device, copy=True) if torch.is_tensor(v) else v
                                          for k, v in loaded["state"][i].items()}

        # after the caller's hooks before the load, which may replace the dictionary, and before those after it
        hooks = (self.register_load_state_dict_pre_hook(lambda optimizer, given: loaded.update(given)),
                 self.register_load_state_dict_post_hook(restore, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
