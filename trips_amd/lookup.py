"""Lookups in a table of descriptors by index, with scaling, and their gradient in the order of the indexes, over the HIP
kernels of include/trips_lookup.h.

A scene's texture [C,T] read by t_index (which the splat otherwise does inside its kernels, and whose gradient the splat
adds up with atomics where points share a texel), or any other table of learned rows. The gradient of a shared entry is
summed in the order of its points: the same bits every time.
"""
import torch
from torch.autograd.function import once_differentiable

from . import abi
from .renderer import get_context

COLUMNS, ROWS = abi.TRIPS_TABLE_COLUMNS, abi.TRIPS_TABLE_ROWS
_DTYPES = {torch.float32: abi.TRIPS_DTYPE_F32, torch.bfloat16: abi.TRIPS_DTYPE_BF16, torch.float16: abi.TRIPS_DTYPE_F16}
_INDEX_DTYPES = {torch.int32: abi.TRIPS_INDEX_I32, torch.int64: abi.TRIPS_INDEX_I64}


def _check_index(index):
    if index.dtype not in _INDEX_DTYPES:
        raise ValueError(f"index: int32 or int64 expected, got {index.dtype}")
    if index.device.type != "cuda":
        raise RuntimeError("lookups need tensors on a GPU: there is no CPU implementation")


def _rows_of(name, t, device):
    """t [A, B] with adjacent elements in a row, and the distance of its rows."""
    if t.dim() != 2 or t.dtype not in _DTYPES or t.device != device:
        raise ValueError(f"{name}: a float32, bfloat16 or float16 matrix on the index's device expected, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    if (t.stride(1) != 1 and t.shape[1] > 1) or t.stride(0) < 0:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _desc(layout, dtype, index_dtype, texels, points, channels, table_stride, values_stride, scale, accumulate=False):
    return abi.TripsLookupDesc(abi.TRIPS_ABI_VERSION, layout, _DTYPES[dtype], _INDEX_DTYPES[index_dtype], texels, points, channels,
                               int(accumulate), table_stride, values_stride, scale)


def _check_layout(layout):
    if layout not in (COLUMNS, ROWS):
        raise ValueError(f"layout: COLUMNS or ROWS expected, got {layout!r}")


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
        if own is not None and (own.data_ptr() != index.data_ptr() or own.dtype != index.dtype or own.stride() != index.stride()
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


@torch.no_grad()
def lookup_plan(index, num_texels):
    """The order of the points by their texel. Indexes outside [0, num_texels) come last and count for no texel."""
    _check_index(index)
    if num_texels < 0:
        raise ValueError(f"num_texels = {num_texels}")
    ctx = get_context(index.device)
    order = torch.empty(index.numel(), dtype=torch.int32, device=index.device)
    starts = torch.empty(num_texels + 1, dtype=torch.int32, device=index.device)
    ctx.lookup_plan(num_texels, index.contiguous(), _INDEX_DTYPES[index.dtype], order, starts)
    return LookupPlan(order, starts, index)


def _forward(table, index, scale, layout):
    table, stride = _rows_of("table", table, index.device)
    columns = layout == COLUMNS
    channels, texels = (table.shape[0], table.shape[1]) if columns else (table.shape[1], table.shape[0])
    points = index.numel()
    values = torch.empty((channels, points) if columns else (points, channels), dtype=table.dtype, device=index.device)
    if channels and points:
        desc = _desc(layout, table.dtype, index.dtype, texels, points, channels, stride, values.shape[1], scale)
        get_context(index.device).lookup_forward(desc, table, index.contiguous(), values)
    return values


@torch.no_grad()
def lookup_backward(grad, index, num_texels, scale=1.0, layout=COLUMNS, plan=None, out=None):
    """The table's gradient from that of its looked-up values: [C, T] from [C, N], or [T, C] from [N, C]. plan: lookup_plan of the
    index, where a program keeps it (it is made here otherwise). out: a table gradient to add to, instead of a new one."""
    _check_layout(layout)
    _check_index(index)
    grad, grad_stride = _rows_of("grad", grad, index.device)
    columns = layout == COLUMNS
    channels, points = (grad.shape[0], grad.shape[1]) if columns else (grad.shape[1], grad.shape[0])
    if points != index.numel():
        raise ValueError(f"grad: {points} points, index has {index.numel()}")
    if plan is None:
        plan = lookup_plan(index, num_texels)
    plan.check(index, num_texels)
    shape = (channels, num_texels) if columns else (num_texels, channels)
    if out is None:
        d_table, accumulate = torch.empty(shape, dtype=grad.dtype, device=grad.device), False
    else:
        if tuple(out.shape) != shape or out.dtype != grad.dtype or out.device != grad.device or (out.stride(1) != 1 and shape[1] > 1) \
                or (shape[0] > 1 and out.stride(0) < shape[1]):
            raise ValueError(f"out: a {grad.dtype} tensor {shape} with adjacent elements in a row expected")
        d_table, accumulate = out, True
    if channels and num_texels:
        desc = _desc(layout, grad.dtype, index.dtype, num_texels, points, channels, d_table.stride(0) if shape[0] > 1 else shape[1],
                     grad_stride, scale, accumulate)
        get_context(index.device).lookup_backward(desc, grad, plan.order, plan.starts, d_table)
    return d_table


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, layout, plan):
        ctx.save_for_backward(index)
        ctx.args = (table.shape[1] if layout == COLUMNS else table.shape[0], scale, layout, plan)
        return _forward(table, index, scale, layout)

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
    _check_layout(layout)
    _check_index(index)
    if table.dim() != 2:
        raise ValueError(f"table: a matrix expected, got {tuple(table.shape)}")
    if plan is not None:
        plan.check(index, table.shape[1] if layout == COLUMNS else table.shape[0])
    if torch.is_grad_enabled() and table.requires_grad:
        return _Lookup.apply(table, index, float(scale), layout, plan)
    return _forward(table.detach(), index, scale, layout)
