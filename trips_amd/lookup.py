"""Lookups in a table of descriptors by index, with scaling, and their gradient in the order of the indexes, over the HIP
kernels of include/trips_lookup.h.

A scene's texture [C,T] read by t_index (which the splat otherwise does inside its kernels, and whose gradient the splat
adds up with atomics where points share a texel), or any other table of learned rows. The gradient of a shared entry is
summed in the order of its points: the same bits every time.
"""
import contextlib

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import abi
from ._host import host as _host
from .renderer import _stream_ptr, _untraced, get_context

COLUMNS, ROWS = abi.TRIPS_TABLE_COLUMNS, abi.TRIPS_TABLE_ROWS


def _where(index):
    """The context of the index's device and its current stream, as the extension takes them (it refuses other devices)."""
    if index.device.type != "cuda":
        return 0, 0
    ctx = get_context(index.device)
    return ctx.ctx.value, _stream_ptr(ctx.device)


def _needs_function(table, index):
    """Whether torch has to see a lookup: to record it (a graph, a trace) or to refuse it (forward-mode duals, a functional
    transform that follows one of the tensors). The kernels' call by itself would lose the derivative, or leave a trace a constant."""
    return (table.requires_grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0 or torch.jit.is_tracing() or _transformed(table, index)


def _transformed(*tensors):
    if not torch._C._are_functorch_transforms_active():
        return False
    return any(torch._C._functorch.is_functorch_wrapped_tensor(t) or torch._C._functorch.is_functionaltensor(t) for t in tensors)


def _refuse_unseen(what, *tensors):
    """For what has no autograd function: nothing is computed that torch would take for something else."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} is not recorded by a trace: call it before")
    if _transformed(*tensors):
        raise RuntimeError(f"{what} of tensors that a functional transform follows is not supported")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _version(index):
    return None if index is None or index.is_inference() else index._version


class LookupPlan:
    """The points of an index in the order of their texels: order [N] and starts [T + 1] (int32; see trips_lookup_plan).
    It belongs to the index that it was made of, as it was then; made in a capture, it holds nothing before the first replay."""

    def __init__(self, order, starts, index=None):
        if order.dtype != torch.int32 or starts.dtype != torch.int32 or not order.is_contiguous() or not starts.is_contiguous() \
                or order.device != starts.device or starts.numel() < 1:
            raise ValueError("a plan is two contiguous int32 tensors: order [N] and starts [T + 1]")
        self.order, self.starts = order, starts
        self.index = index
        self._own = None
        self.version = _version(index)

    def __getstate__(self):
        # (a copy of the index counts its versions anew: what goes along is whether the index is still what the plan was made of)
        return {**self.__dict__, "version": _version(self.index) == self.version}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.version = _version(self.index) if state["version"] else -1

    def check(self, index, texels):
        if self.order.numel() != index.numel() or self.starts.numel() != texels + 1 or self.order.device != index.device:
            raise ValueError(f"the plan is for {self.order.numel()} points and {self.starts.numel() - 1} texels, not for "
                             f"{index.numel()} and {texels}")
        own = self.index
        if own is not None and (own.data_ptr() != index.data_ptr() or own.dtype != index.dtype
                                or ((own.stride() != index.stride() or own.shape != index.shape) and not (own.is_contiguous() and index.is_contiguous()))
                                or _version(index) != self.version):
            raise ValueError("the plan was made of another index, or the index was changed since")

    def keep_own_index(self):
        """Makes own_index() of the plan's index, on the current stream, like the plan itself, for all that use the plan."""
        if self.index is None:
            raise ValueError("the plan was made without an index")
        self._own = own_index(self.index, self.starts.numel() - 1)

    def own_index(self, index):
        """own_index() of the plan's index: the one that keep_own_index() made, or a new one (a call that made and kept it on the way
        would leave it to others before its capture was replayed, or to another stream before it was written)."""
        self.check(index, self.starts.numel() - 1)
        return own_index(index, self.starts.numel() - 1) if self._own is None else self._own


def own_index(index, num_texels):
    """The number of each point, -1 where its index is outside [0, num_texels): int32, in the index's shape."""
    own = torch.arange(index.numel(), dtype=torch.int32, device=index.device).reshape(index.shape)
    return torch.where((index >= 0) & (index < num_texels), own, -1)


def lookup_plan(index, num_texels):
    """The order of the points by their texel. Indexes outside [0, num_texels) come last and count for no texel."""
    _refuse_unseen("lookup_plan", index)
    return LookupPlan(*_host().lookup_plan(*_where(index), index, num_texels), index)


def lookup_backward(grad, index, num_texels, scale=1.0, layout=COLUMNS, plan=None, out=None):
    """The table's gradient from that of its looked-up values: [C, T] from [C, N], or [T, C] from [N, C]. plan: lookup_plan of the
    index, where a program keeps it (it is made here otherwise). out: a table gradient to add to, instead of a new one."""
    if plan is not None:
        plan.check(index, num_texels)
    order, starts = (None, None) if plan is None else (plan.order, plan.starts)
    return _table_gradient(grad, index, order, starts, num_texels, scale, layout, out)


def _table_gradient(grad, index, order, starts, num_texels, scale, layout, out=None):
    _refuse_unseen("lookup_backward", grad, index)
    return _host().lookup_backward(*_where(index), grad.detach(), index, order, starts, num_texels, scale, layout, out)


def _check_plan(table, index, layout, plan):
    if plan is not None and table.dim() == 2:
        plan.check(index, table.shape[1] if layout == COLUMNS else table.shape[0])


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, layout, plan):
        # The plan is checked here for a trace, which may be run with another index; what a trace sees of a function is its call alone.
        with _untraced() if torch.jit.is_tracing() else contextlib.nullcontext():
            _check_plan(table, index, layout, plan)
            values = _host().lookup(*_where(index), table.detach(), index, scale, layout)
        # The plan's tensors are saved like the index, so that the gradient is of the lookup that was made: hooks on what is saved may hand
        # back other tensors, and one that was written to meanwhile is refused. (Those of inference mode cannot be saved, or written to here.)
        order, starts = (None, None) if plan is None else (plan.order, plan.starts)
        saved = plan is not None and not (order.is_inference() or starts.is_inference())
        ctx.save_for_backward(index, *((order, starts) if saved else ()))
        ctx.args = (table.shape[1] if layout == COLUMNS else table.shape[0], scale, layout)
        ctx.plan = None if saved else (order, starts)
        return values

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        index, *plan = ctx.saved_tensors
        return _table_gradient(grad, index, *(ctx.plan or plan), *ctx.args), None, None, None, None


def lookup(table, index, scale=1.0, layout=COLUMNS, plan=None):
    """scale times the entries of the table that the index names: [C, N] from a table [C, T] (COLUMNS, a scene's texture), or
    [N, C] from [T, C] (ROWS); N = index.numel(). Zeros where an index is outside the table (padding). Differentiable in the
    table; plan: lookup_plan of the index, for the gradient, where a program keeps it."""
    if _needs_function(table, index):
        return _Lookup.apply(table, index, scale, layout, plan)
    _check_plan(table, index, layout, plan)
    return _host().lookup(*_where(index), table.detach(), index, scale, layout)
