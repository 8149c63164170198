"""AdamW over dense parameters and the global norm of gradients, over the HIP kernels of include/trips_optim.h.

For what MyAdam's rules do not suit: the reconstruction net (which the reference steps with libtorch's optimiser,
src/lib/models/Pipeline.cpp:870-882) and any other tensor whose every element is stepped every time. All tensors of one
combination of types go through one launch per 40 of them; clipping by the global norm stays on the device, and so do the
step counts, so that a step may be captured into a HIP graph.

A graph's backward pass must not be captured while an eager graph of the same leaves is alive (torch ends the process).
"""
import math
import struct

import torch
from torch.autograd import _profiler_enabled
from torch.autograd.graph import increment_version as _increment_version
from torch.optim import optimizer as _optimizer

from . import abi
from .renderer import get_context

_DTYPES = {torch.float32: abi.TRIPS_DTYPE_F32, torch.bfloat16: abi.TRIPS_DTYPE_BF16, torch.float16: abi.TRIPS_DTYPE_F16}
_pack_tensor, _pack_options = struct.Struct("8Qq4i").pack, struct.Struct("5d").pack  # TripsAdamWTensor up to `lr`, and from there
_pack_grad = struct.Struct("Qqi4x").pack                                             # TripsGradTensor
_MOMENTS = {8: (torch.float8_e4m3fn, torch.float8_e5m2), 32: (torch.float32, torch.float32)}


def _contiguous(g):
    if g.is_sparse:
        _refuse(None, g, 0)
    return g.detach().contiguous()


def _refuse(p, g, device):
    """Says what is wrong with a parameter (or None) and its gradient."""
    if g.is_sparse:
        raise RuntimeError("sparse gradients are not supported")
    if g.dtype not in _DTYPES:
        raise RuntimeError(f"gradients are float32, bfloat16 or float16, not {g.dtype}")
    if p is not None and (p.dtype not in _DTYPES or not p.is_contiguous()):
        raise RuntimeError("AdamW needs contiguous float32, bfloat16 or float16 parameters")
    if p is not None and g.numel() != p.numel():
        raise RuntimeError(f"a gradient of {g.numel()} elements for a parameter of {p.numel()}")
    if device < 0:
        raise RuntimeError("the kernels need tensors on a GPU: there is no CPU implementation")
    raise RuntimeError("all tensors of a call must be on one device")


def grad_norm(grads, max_norm=0.0, loss_scale=1.0):
    """[norm, factor] of a list of gradients as a float32 tensor on their device: the root of the sum of all their squares
    divided by loss_scale, and what gradients are multiplied by to undo loss_scale and to clip their norm at max_norm
    (0: no clipping); the factor is NaN where the norm is not finite. Nothing is read back. AdamW.step() takes it as `grad_norm`."""
    table, temporary, device = [], [], None
    for g in grads:
        dtype, index = _DTYPES.get(g.dtype), g.get_device()
        if device is None:
            device = index
        if dtype is None or index < 0 or index != device:
            _refuse(None, g, device)
        if not g.is_contiguous():
            g = _contiguous(g)
            temporary.append(g)
        table.append(_pack_grad(g.data_ptr(), g.numel(), dtype))
    if not table:
        raise ValueError("grad_norm of no gradients")
    ctx = get_context(device)
    device = ctx.device
    out = torch.empty(2, dtype=torch.float32, device=device)
    ctx.grad_norm(b"".join(table), len(table), max_norm, loss_scale, out, ctx.alloc_bytes(abi.TRIPS_GRAD_NORM_WORKSPACE_BYTES))
    return out


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay: parameters float32, bfloat16 or float16, moments in 32 or in 8 bits.

    state_bits 8 holds the moments as 8-bit floats with a scale per 256 elements, rounded stochastically (`seed`; see
    TripsAdamWTensor in include/trips_optim.h), in parameters of at least min_8bit_size elements. max_grad_norm clips the
    global norm of all gradients; with it, or with skip_nonfinite, a step whose gradients are not all finite is skipped on the
    device: parameters, state and step counts stay as they are. loss_scale: what the loss was multiplied by; an attribute, like
    max_grad_norm, that may be changed between steps. After a step `grad_norm` holds [norm, factor] (a device tensor, written
    over by the next step) if it was computed.

    State per parameter: step (int32, on the device), first_moment, second_moment, and with 8 bits first_scale and second_scale;
    moments() gives the moments as numbers. A captured step replays with the learning rates of its capture; a step that is
    captured must not be the first (which makes the state)."""

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
        if state_bits not in _MOMENTS:
            raise ValueError(f"state_bits must be 32 or 8, not {state_bits}")
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
        self._copies = {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size))

    def set_copy(self, p, copy):
        """Every step writes the new value of parameter `p` to `copy` as well (a contiguous tensor of its size, in any of the
        three types), before it is rounded to p's own type. None ends that."""
        if copy is None:
            self._copies.pop(p, None)
            return
        if copy.dtype not in _DTYPES or copy.numel() != p.numel() or not copy.is_contiguous() or copy.device != p.device:
            raise ValueError("a copy is a contiguous float32, bfloat16 or float16 tensor of its parameter's size, on its device")
        self._copies[p] = copy

    def _make_state(self, p, group):
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
        # (An attribute or a call costs 50 to 100 ns, of which a tensor takes a score; what a check finds is said in _refuse.)
        table, params, temporary, device, copies, states, dtypes = [], [], [], None, self._copies, self.state, _DTYPES
        for group in self.param_groups:
            options = _pack_options(group["lr"], *group["betas"], group["eps"], group["weight_decay"])
            for p in group["params"]:
                g = p.grad if grads is None else grads.get(p)
                if g is None:
                    continue
                n, index = p.numel(), p.get_device()
                weight_dtype, grad_dtype = dtypes.get(p.dtype), dtypes.get(g.dtype)
                if device is None:
                    device = index
                if weight_dtype is None or grad_dtype is None or index < 0 or index != device or g.get_device() != index \
                        or g.numel() != n or not p.is_contiguous():
                    _refuse(p, g, device)
                if not g.is_contiguous():
                    g = _contiguous(g)
                    temporary.append(g)
                st = states.get(p) or self._make_state(p, group)
                if "first_scale" in st:
                    first_scale, second_scale, bits = st["first_scale"].data_ptr(), st["second_scale"].data_ptr(), 8
                else:
                    first_scale, second_scale, bits = 0, 0, 32
                copy_at, copy_dtype = 0, 0
                if copies:
                    copy = copies.get(p)
                    if copy is not None:
                        copy_at, copy_dtype = copy.data_ptr(), dtypes[copy.dtype]
                params.append(p)
                table += (_pack_tensor(p.data_ptr(), g.data_ptr(), st["first_moment"].data_ptr(), st["second_moment"].data_ptr(),
                                       first_scale, second_scale, copy_at, st["step"].data_ptr(), n, weight_dtype, grad_dtype,
                                       copy_dtype, bits), options)
        if not params:
            return loss
        ctx = get_context(device)
        if self._workspace is None or self._workspace.device != ctx.device or self._workspace_for < len(params):
            self._workspace = ctx.alloc_bytes(ctx.adamw_workspace_size(len(params)))
            self._workspace_for = len(params)
            self._norm = torch.empty(2, dtype=torch.float32, device=ctx.device)
        max_norm = self.max_grad_norm or 0.0
        compute = grad_norm is None and (max_norm > 0 or self.skip_nonfinite)
        if grad_norm is not None and (grad_norm.dtype != torch.float32 or grad_norm.numel() != 2 or grad_norm.device != ctx.device
                                      or not grad_norm.is_contiguous()):
            raise ValueError("grad_norm: two float32 numbers on the parameters' device expected")
        self.grad_norm = self._norm if compute else grad_norm
        options = abi.TripsAdamWOptions(abi.TRIPS_ABI_VERSION, self.seed & 0xFFFFFFFF,
                                        None if self.grad_norm is None else self.grad_norm.data_ptr(), int(compute),
                                        max_norm if compute else 0.0, self.loss_scale)
        ctx.adamw_step(b"".join(table), len(params), options, self._workspace)
        _increment_version(params)  # (a backward pass that needs the old values raises)
        return loss

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

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # (the base class casts state to the parameters' type: here it keeps its own)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            st = state_dict["state"].get(i)
            if st is not None:
                self.state[p] = {k: v.detach().to(p.device).clone() if torch.is_tensor(v) else v for k, v in st.items()}


_watched_step = torch.optim.Optimizer.profile_hook_step(AdamW._step)
