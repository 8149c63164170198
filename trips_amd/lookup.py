"""Lookups in a table of descriptors by index, with scaling, and their gradient in the order of the indexes, over the HIP
kernels of include/trips_lookup.h.

A scene's texture [C,T] read by t_index (which the splat otherwise does inside its kernels, and whose gradient the splat
adds up with atomics where points share a texel), or any other table of learned rows. The gradient of a shared entry is
summed in the order of its points: the same bits every time.
"""
import torch
from torch.autograd.function import once_differentiable

from . import abi
from ._host import host as _host
from .renderer import _stream_ptr, get_context

COLUMNS, ROWS = abi.TRIPS_TABLE_COLUMNS, abi.TRIPS_TABLE_ROWS


def _where(index):
    """The context of the index's device and its current stream, as the extension takes them (it refuses other devices)."""
    if index.device.type != "cuda":
        return 0, 0
    ctx = get_context(index.device)
    return ctx.ctx.value, _stream_ptr(ctx.device)


class LookupPlan:
    """The points of an index in the order of their texels: order [N] and starts [T + 1] (int32; see trips_lookup_plan).
    It belongs to the index that it was made of, as it was then."""

    def __init__(self, order, starts, index=None):
        if order.dtype != torch.int32 or starts.dtype != torch.int32 or not order.is_contiguous() or not starts.is_contiguous() \
                or order.device != starts.device or starts.numel() < 1:
            raise ValueError("a plan is two contiguous int32 tensors: order [N] and starts [T + 1]")
        self.order, self.starts = order, starts
        self.index = index
        self._own = None
        self.version = None if index is None or index.is_inference() else index._version

    def check(self, index, texels):
        if self.order.numel() != index.numel() or self.starts.numel() != texels + 1 or self.order.device != index.device:
            raise ValueError(f"the plan is for {self.order.numel()} points and {self.starts.numel() - 1} texels, not for "
                             f"{index.numel()} and {texels}")
        own = self.index
        if own is not None and (own.data_ptr() != index.data_ptr() or own.dtype != index.dtype
                                or (own.stride() != index.stride() and not (own.is_contiguous() and index.is_contiguous()))
                                or (None if index.is_inference() else index._version) != self.version):
            raise ValueError("the plan was made of another index, or the index was changed since")

    def own_index(self, index):
        """own_index() of the plan's index, made once."""
        self.check(index, self.starts.numel() - 1)
        if self._own is None:
            self._own = own_index(index, self.starts.numel() - 1)
        return self._own


def own_index(index, num_texels):
    """The number of each point, -1 where its index is outside [0, num_texels): int32, in the index's shape."""
    own = torch.arange(index.numel(), dtype=torch.int32, device=index.device).reshape(index.shape)
    return torch.where((index >= 0) & (index < num_texels), own, -1)


def lookup_plan(index, num_texels):
    """The order of the points by their texel. Indexes outside [0, num_texels) come last and count for no texel."""
    return LookupPlan(*_host().lookup_plan(*_where(index), index, num_texels), index)


def lookup_backward(grad, index, num_texels, scale=1.0, layout=COLUMNS, plan=None, out=None):
    """The table's gradient from that of its looked-up values: [C, T] from [C, N], or [T, C] from [N, C]. plan: lookup_plan of the
    index, where a program keeps it (it is made here otherwise). out: a table gradient to add to, instead of a new one."""
    if plan is not None:
        plan.check(index, num_texels)
    order, starts = (None, None) if plan is None else (plan.order, plan.starts)
    return _host().lookup_backward(*_where(index), grad.detach(), index, order, starts, num_texels, scale, layout, out)


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, layout, plan):
        values = _host().lookup(*_where(index), table.detach(), index, scale, layout)
        ctx.save_for_backward(index)
        ctx.args = (table.shape[1] if layout == COLUMNS else table.shape[0], scale, layout, plan)
        return values

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        index, = ctx.saved_tensors
        texels, scale, layout, plan = ctx.args
        return lookup_backward(grad, index, texels, scale, layout, plan), None, None, None, None


def lookup(table, index, scale=1.0, layout=COLUMNS, plan=None):
    """scale times the entries of the table that the index names: [C, N] from a table [C, T] (COLUMNS, a scene's texture), or
    [N, C] from [T, C] (ROWS); N = index.numel(). Zeros where an index is outside the table (padding). Differentiable in the
    table; plan: lookup_plan of the index, for the gradient, where a program keeps it."""
    if plan is not None and table.dim() == 2:
        plan.check(index, table.shape[1] if layout == COLUMNS else table.shape[0])
    if table.requires_grad and torch.is_grad_enabled():
        return _Lookup.apply(table, index, scale, layout, plan)
    return _host().lookup(*_where(index), table.detach(), index, scale, layout)
