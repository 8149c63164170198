"""AdamW over dense parameters and the global norm of gradients, over the HIP kernels of include/trips_optim.h.

For what MyAdam's rules do not suit: the reconstruction net (which the reference steps with libtorch's optimiser,
src/lib/models/Pipeline.cpp:870-882) and any other tensor whose every element is stepped every time. All tensors of one
combination of types go through one launch, after a small one per 40 of them; clipping by the global norm stays on the
device, and so do the step counts, so that a step may be captured into a HIP graph.

A graph's backward pass must not be captured while an eager graph of the same leaves is alive (torch ends the process).
"""
import math

import torch
from torch.autograd import _profiler_enabled
from torch.optim import optimizer as _optimizer

from . import _lib, abi
from ._host import host as _host
from .renderer import _stream_ptr, get_context

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_MOMENTS = {8: (torch.float8_e4m3fn, torch.float8_e5m2), 32: (torch.float32, torch.float32)}


def grad_norm(grads, max_norm=0.0, loss_scale=1.0):
    """[norm, factor] of a list of gradients as a float32 tensor on their device: the root of the sum of all their squares
    divided by loss_scale, and what gradients are multiplied by to undo loss_scale and to clip their norm at max_norm
    (0: no clipping); the factor is NaN where the norm is not finite. Nothing is read back. AdamW.step() takes it as `grad_norm`."""
    table = _host().NormTable()
    count, device = table.collect(grads)
    if not count:
        raise ValueError("grad_norm of no gradients")
    ctx = get_context(device)
    out = torch.empty(2, dtype=torch.float32, device=ctx.device)
    _lib.check(table.norm(ctx.ctx.value, max_norm, loss_scale, out, ctx.alloc_bytes(abi.TRIPS_GRAD_NORM_WORKSPACE_BYTES),
                          _stream_ptr(ctx.device)))
    return out


def _check_bits(bits):
    if bits not in _MOMENTS:
        raise ValueError(f"state_bits must be 32 or 8, not {bits}")


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay: parameters float32, bfloat16 or float16, moments in 32 or in 8 bits.

    state_bits 8 holds the moments as 8-bit floats with a scale per 256 elements, rounded stochastically (`seed`; see
    TripsAdamWTensor in include/trips_optim.h), in parameters of at least min_8bit_size elements. max_grad_norm clips the
    global norm of all gradients; with it, or with skip_nonfinite, a step whose gradients are not all finite is skipped on the
    device: parameters, state and step counts stay as they are. loss_scale: what the loss was multiplied by; an attribute, like
    max_grad_norm, that may be changed between steps. After a step `grad_norm` holds [norm, factor] (a device tensor, written
    over by the next step) if it was computed.

    State per parameter: step (int32, on the device), first_moment, second_moment, and with 8 bits first_scale and second_scale;
    moments() gives the moments as numbers. A captured step replays with the learning rates and goes on with the moments of its
    capture: after load_state_dict() it has to be captured anew. A parameter's first step, which makes its state, cannot be
    captured. Steps of one optimiser must not overlap, and the optimiser has to outlive the graphs that hold its steps."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, min_8bit_size=4096,
                 max_grad_norm=0.0, skip_nonfinite=False, loss_scale=1.0, seed=0):
        if not 0 <= lr < math.inf:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0 <= eps < math.inf:
            raise ValueError(f"Invalid epsilon value: {eps}")
        for i, beta in enumerate(betas):
            if not 0 <= beta < 1.0:
                raise ValueError(f"Invalid beta parameter at index {i}: {beta}")
        if not 0 <= weight_decay < math.inf:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        _check_bits(state_bits)
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        if not 0 < loss_scale < math.inf:
            raise ValueError(f"Invalid loss_scale: {loss_scale}")
        self.max_grad_norm = max_grad_norm
        self.skip_nonfinite = skip_nonfinite
        self.loss_scale = loss_scale
        self.seed = seed
        self.grad_norm = None
        self._workspace = None
        self._kept = []  # what captured steps write and later ones do not
        self._captured = False
        self._copies = {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size))

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):  # (the base class refuses others)
            _check_bits(param_group.get("state_bits", self.defaults["state_bits"]))
        super().add_param_group(param_group)
        params = self.param_groups[-1]["params"]
        if len(set(params)) != len(params):  # (of which the base class only warns; one in two groups it refuses)
            del self.param_groups[-1]
            raise ValueError("a parameter is in its group twice: its steps would run side by side")

    def set_copy(self, p, copy):
        """Every step writes the new value of parameter `p` to `copy` as well (a contiguous tensor of its size, in any of the
        three types), before it is rounded to p's own type. None ends that. A copied or unpickled optimiser has no copies yet."""
        if copy is None:
            self._copies.pop(p, None)
            return
        if copy.dtype not in _DTYPES or copy.numel() != p.numel() or not copy.is_contiguous() or copy.device != p.device:
            raise ValueError("a copy is a contiguous float32, bfloat16 or float16 tensor of its parameter's size, on its device")
        self._copies[p] = copy

    def _make_state(self, p, group):
        _check_bits(group["state_bits"])
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a parameter's first step makes its state and cannot be captured into a graph")
        bits = 8 if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"] else 32
        first, second = _MOMENTS[bits]
        st = self.state[p]
        st["step"] = torch.zeros((), dtype=torch.int32, device=p.device)
        st["first_moment"] = torch.zeros(p.shape, dtype=first, device=p.device)
        st["second_moment"] = torch.zeros(p.shape, dtype=second, device=p.device)
        if bits == 8:
            blocks = -(-p.numel() // abi.TRIPS_MOMENT_BLOCK)
            st["first_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
            st["second_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        return st

    def step(self, closure=None, grads=None, grad_norm=None):
        """grads: {parameter: gradient}, for gradients in another type than their parameter's, instead of the parameters' own;
        grad_norm: the [norm, factor] to go by, where this optimiser's gradients are only some of those whose norm counts."""
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _optimizer._global_optimizer_pre_hooks \
                or _optimizer._global_optimizer_post_hooks or _profiler_enabled():
            return _watched_step(self, closure, grads, grad_norm)
        return self._step(closure, grads, grad_norm)

    # The base class would wrap step() for its hooks and the profiler's range: some 10 us a step, as much as the kernels take of
    # a small net's. Here that way is gone where there is something to call.
    step.hooked = True

    def _step(self, closure, grads, grad_norm):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        table = _host().StepTable()
        count, device = table.collect(self.param_groups, self.state, self._copies, grads, self._make_state)
        if not count:
            return loss
        ctx = get_context(device)
        if self._workspace is None or self._workspace.device != ctx.device or self._workspace_for < count:
            self._make_workspace(ctx)
        stream = _stream_ptr(ctx.device)
        if stream not in self._streams:  # (its memory is not to be given away before this stream is done with it)
            for t in (self._workspace, self._norm):
                t.record_stream(torch.cuda.current_stream(ctx.device))
            self._streams.add(stream)
        self._captured = self._captured or torch.cuda.is_current_stream_capturing()
        max_norm = self.max_grad_norm or 0.0
        compute = grad_norm is None and (max_norm > 0 or self.skip_nonfinite)
        if grad_norm is not None and (grad_norm.dtype != torch.float32 or grad_norm.numel() != 2 or grad_norm.device != ctx.device
                                      or not grad_norm.is_contiguous()):
            raise ValueError("grad_norm: two float32 numbers on the parameters' device expected")
        self.grad_norm = self._norm if compute else grad_norm
        _lib.check(table.step(ctx.ctx.value, self.seed & 0xFFFFFFFF, self.grad_norm, compute, max_norm if compute else 0.0, self.loss_scale,
                              self._workspace, stream))
        return loss

    def _make_workspace(self, ctx):
        # For all parameters, whichever have a gradient this time. What an earlier one was captured with stays alive with it.
        if self._workspace is not None:
            self._kept.append((self._workspace, self._norm))
        self._workspace_for = sum(len(g["params"]) for g in self.param_groups)
        self._workspace = ctx.alloc_bytes(ctx.adamw_workspace_size(self._workspace_for))
        self._norm = torch.empty(2, dtype=torch.float32, device=ctx.device)
        self._streams = {_stream_ptr(ctx.device)}

    _OWN = ("max_grad_norm", "skip_nonfinite", "loss_scale", "seed")

    def __getstate__(self):
        return {**super().__getstate__(), **{k: getattr(self, k) for k in self._OWN}}

    def __setstate__(self, state):
        # Of an optimiser that is being copied or unpickled, which has none of these yet: a workspace of its own, and no copies
        # of its parameters. load_state_dict() ends here as well, where what there is stays.
        for name, value in (("grad_norm", None), ("_workspace", None), ("_kept", []), ("_captured", False), ("_copies", {})):
            self.__dict__.setdefault(name, value)
        super().__setstate__(state)

    @torch.no_grad()
    def moments(self, p):
        """First and second moment of a parameter as float32 tensors of its shape."""
        st = self.state[p]
        first, second = st["first_moment"], st["second_moment"]
        if "first_scale" not in st:
            return first.clone(), second.clone()

        def numbers(codes, scale):
            wide = scale.repeat_interleave(abi.TRIPS_MOMENT_BLOCK)[:codes.numel()]
            return (codes.reshape(-1).to(torch.float32) * wide).reshape(codes.shape)
        return numbers(first, st["first_scale"]), numbers(second, st["second_scale"])

    def state_dict(self):
        """The base class's, and under "options" what belongs to the optimiser and not to a group: max_grad_norm, skip_nonfinite,
        loss_scale and seed. load_state_dict() takes them where they are there."""
        return {**super().state_dict(), "options": {k: getattr(self, k) for k in self._OWN}}

    def load_state_dict(self, state_dict):
        # The base class would cast the state to the parameters' types. It loads all else here; the state itself, in its own types,
        # goes in between the hooks: those before have made the dict what it is, those behind find it loaded.
        loaded, ids, before = {}, [], dict(self.state)

        def behind_pre_hooks(_, final):
            loaded.update(final)
            ids.extend(i for g in final["param_groups"] for i in g["params"])
            known = set(ids)
            return {**final, "state": {k: v for k, v in final["state"].items() if k not in known}}

        def before_post_hooks(_):
            if self._captured:  # (a graph goes on writing to the state of its capture)
                self._kept.append(before)
                self._captured = False
            for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
                if i in loaded["state"]:
                    self.state[p] = {k: v.detach().to(p.device).clone(memory_format=torch.contiguous_format) if torch.is_tensor(v) else v
                                     for k, v in loaded["state"][i].items()}
            for k, v in loaded.get("options", {}).items():
                if k in self._OWN:
                    setattr(self, k, v)
        handles = (self.register_load_state_dict_pre_hook(behind_pre_hooks),
                   self.register_load_state_dict_post_hook(before_post_hooks, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()


_watched_step = torch.optim.Optimizer.profile_hook_step(AdamW._step)
