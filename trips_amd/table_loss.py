"""Softmax cross entropy of rows against all entries of a table, and its gradients, over the HIP kernels of include/trips_loss.h.

The other end of a table whose rows lookup() reads: which entry a row belongs to, among all of them. The logits are never kept:
the loss is made in one pass over the table, the gradients from logits that are computed again in pieces of it.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import abi
from ._host import host as _host
from .lookup import _transformed, _where
from .renderer import _untraced

REDUCTIONS = {"none": abi.TRIPS_REDUCE_NONE, "sum": abi.TRIPS_REDUCE_SUM, "mean": abi.TRIPS_REDUCE_MEAN}


class _TableCrossEntropy(torch.autograd.Function):
    """For modes that have to see a call: traces record it, forward-mode levels and functional transforms refuse it."""
    @staticmethod
    def forward(ctx, rows, table, target, scale, reduction):
        with _untraced():
            loss, kept = _host().table_loss(*_where(target), rows.detach(), table.detach(), target, scale, reduction)
        ctx.save_for_backward(table, kept)
        ctx.args = (rows.shape[0], scale, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        table, kept = ctx.saved_tensors
        d_rows, d_table = _host().table_loss_backward(*_where(kept), grad, table.detach(), kept, *ctx.args, *ctx.needs_input_grad[:2])
        return d_rows, d_table, None, None, None


def table_cross_entropy(rows, table, target, scale=1.0, reduction="mean"):
    """What rows [N, C] lose on their targets among the entries of table [T, C]: with logits l = scale <row, entry>, the log of
    the sum of exp(l) over all entries, minus l of the target. target: N integers (int32 or int64, of any shape, like an index of
    lookup()); rows whose target is outside the table (padding) count for nothing and get no gradient, whatever they hold.

    The table is of lookup()'s layout ROWS. Rows and tables whose channels are not adjacent in memory, a texture [C, T] turned by t() among them, are copied
    first, in the forward and again in the backward pass; a program that keeps its table as [T, C] has neither copy.

    reduction: "none" gives [N], "sum" and "mean" one number, the mean over the rows that count (0 where none does); float32
    whatever the type of rows and table (float32, bfloat16 or float16, the same of both). Differentiable in rows and table, once, and
    not in scale; gradients have their type. What the gradients need of the rows is a copy of those that count, kept with the graph; they may be written to
    meanwhile, the table may not.

    In 16 bits the losses and the probabilities are made in 32, and what the gradients' products take of a probability is rounded to the type (half a step of it)
    where the problem is large: the gradients are off by 1.1 to 1.8 times what their own rounding takes. Up to 128 rows of a table of 2^22 numbers, and where a table's
    gradient has fewer than 256 tiles of 128 x 128, the rest of it is taken too, which large problems would pay half as much time again for. In float16 the gradients of rows
    whose loss counts 2^-15 as much as another's lose precision. Rows and tables in float32 lose nothing of this."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction: 'none', 'sum' or 'mean' expected, got {reduction!r}")
    reduction = REDUCTIONS[reduction]
    followed = (rows, table, target)
    if torch.is_tensor(scale):
        if scale.requires_grad and torch.is_grad_enabled():
            raise ValueError("scale: it gets no gradient; scale the rows where it is learned")
        followed += (scale,)
    if forward_ad._current_level >= 0 or torch.jit.is_tracing() or _transformed(*followed):
        return _TableCrossEntropy.apply(rows, table, target, scale, reduction)
    if torch.is_grad_enabled() and (rows.requires_grad or table.requires_grad):
        ctx, stream = _where(target)
        return _host().table_loss_graph(ctx, stream, rows, table, target, scale, reduction)
    return _host().table_loss(*_where(target), rows.detach(), table.detach(), target, scale, reduction)[0]
