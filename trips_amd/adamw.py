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

from . import abi
from .renderer import get_context

_DTYPES = {torch.float32: abi.TRIPS_DTYPE_F32, torch.bfloat16: abi.TRIPS_DTYPE_BF16, torch.float16: abi.TRIPS_DTYPE_F16}
_pack_tensor = struct.Struct("8Qq4i5d").pack  # TripsAdamWTensor
_pack_grad = struct.Struct("Qqi4x").pack      # TripsGradTensor
_MOMENTS = {8: (torch.float8_e4m3fn, torch.float8_e5m2), 32: (torch.float32, torch.float32)}


def _check_grad(g):
    if g.is_sparse:
        raise RuntimeError("sparse gradients are not supported")
    if g.dtype not in _DTYPES:
        raise RuntimeError(f"gradients are float32, bfloat16 or float16, not {g.dtype}")
    return g if g.is_contiguous() else g.contiguous()


def _device_of(tensors):
    device = tensors[0].device
    if device.type != "cuda":
        raise RuntimeError("the kernels need tensors on a GPU: there is no CPU implementation")
    for t in tensors:
        if t.device != device:
            raise RuntimeError(f"all tensors of a call must be on one device: {t.device} and {device}")
    return device


@torch.no_grad()
def grad_norm(grads, max_norm=0.0, loss_scale=1.0):
    """[norm, factor] of a list of gradients as a float32 tensor on their device: the root of the sum of all their squares
    divided by loss_scale, and what gradients are multiplied by to undo loss_scale and to clip their norm at max_norm
    (0: no clipping); the factor is NaN where the norm is not finite. Nothing is read back. AdamW.step() takes it as `grad_norm`."""
    grads = [_check_grad(g) for g in grads]
    if not grads:
        raise ValueError("grad_norm of no gradients")
    device = _device_of(grads)
    ctx = get_context(device)
    out = torch.empty(2, dtype=torch.float32, device=device)
    table = b"".join([_pack_grad(g.data_ptr(), g.numel(), _DTYPES[g.dtype]) for g in grads])
    ctx.grad_norm(table, len(grads), max_norm, loss_scale, out, ctx.alloc_bytes(abi.TRIPS_ADAMW_WORKSPACE_BYTES))
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

    @torch.no_grad()
    def step(self, closure=None, grads=None, grad_norm=None):
        """grads: {parameter: gradient}, for gradients in another type than their parameter's, instead of the parameters' own;
        grad_norm: the [norm, factor] to go by, where this optimiser's gradients are only some of those whose norm counts."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        table, keep, device = [], [], None
        for group in self.param_groups:
            (beta1, beta2), lr, eps, decay = group["betas"], group["lr"], group["eps"], group["weight_decay"]
            for p in group["params"]:
                g = p.grad if grads is None else grads.get(p)
                if g is None:
                    continue
                weight_dtype = _DTYPES.get(p.dtype)
                if weight_dtype is None or not p.is_contiguous():
                    raise RuntimeError("AdamW needs contiguous float32, bfloat16 or float16 parameters")
                g = _check_grad(g)
                n = p.numel()
                if g.numel() != n:
                    raise RuntimeError(f"a gradient of {g.numel()} elements for a parameter of {n}")
                keep += (p, g)
                st = self.state.get(p) or self._make_state(p, group)
                first, first_scale = st["first_moment"], st.get("first_scale")
                copy = self._copies.get(p) if self._copies else None
                table.append(_pack_tensor(
                    p.data_ptr(), g.data_ptr(), first.data_ptr(), st["second_moment"].data_ptr(),
                    0 if first_scale is None else first_scale.data_ptr(), 0 if first_scale is None else st["second_scale"].data_ptr(),
                    0 if copy is None else copy.data_ptr(), st["step"].data_ptr(), n, weight_dtype, _DTYPES[g.dtype],
                    0 if copy is None else _DTYPES[copy.dtype], 32 if first_scale is None else 8, lr, beta1, beta2, eps, decay))
        if not table:
            return loss
        device = _device_of(keep)
        ctx = get_context(device)
        if self._workspace is None or self._workspace.device != device:
            self._workspace = torch.zeros(abi.TRIPS_ADAMW_WORKSPACE_BYTES, dtype=torch.uint8, device=device)
            self._norm = torch.empty(2, dtype=torch.float32, device=device)
        max_norm = self.max_grad_norm or 0.0
        compute = grad_norm is None and (max_norm > 0 or self.skip_nonfinite)
        if grad_norm is not None and (grad_norm.dtype != torch.float32 or grad_norm.numel() != 2 or grad_norm.device != device
                                      or not grad_norm.is_contiguous()):
            raise ValueError("grad_norm: two float32 numbers on the parameters' device expected")
        self.grad_norm = self._norm if compute else grad_norm
        options = abi.TripsAdamWOptions(abi.TRIPS_ABI_VERSION, self.seed & 0xFFFFFFFF,
                                        None if self.grad_norm is None else self.grad_norm.data_ptr(), int(compute),
                                        max_norm if compute else 0.0, self.loss_scale)
        ctx.adamw_step(b"".join(table), len(table), options, self._workspace)
        return loss

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
