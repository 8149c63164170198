"""Dropout by a counter-based generator, over the HIP kernel of include/trips_loss.h: what is dropped follows from the seed, the
call, the step and an element's place, so the mask is made again for the gradient and never stored, and is the same on every
device, in every type and however the elements are split over launches.
"""
import operator

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._host import host as _host
from .lookup import _transformed, _where
from .renderer import _untraced


def _run(x, p, seed, call, step, residual, want_step):
    number, at = (0, step) if torch.is_tensor(step) else (step, None)
    return _host().dropout(*_where(x), x, p, seed, call, number, at, residual, want_step)


class _Dropout(torch.autograd.Function):
    """For modes that have to see a call: traces record it, forward-mode levels and functional transforms refuse it."""
    @staticmethod
    def forward(ctx, x, p, seed, call, step, residual):
        with _untraced():
            out, used = _run(x.detach(), p, seed, call, step, None if residual is None else residual.detach(), True)
        # (the step may have gone on when the gradient is made: what was used is kept)
        ctx.save_for_backward(*(() if used is None else (used,)))
        ctx.args = (p, seed, call, None if torch.is_tensor(step) else step)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        p, seed, call, step = ctx.args
        d_x = None
        if ctx.needs_input_grad[0]:
            d_x, _ = _run(grad, p, seed, call, ctx.saved_tensors[0] if step is None else step, None, False)
        return d_x, None, None, None, None, grad if ctx.needs_input_grad[5] else None


def dropout(x, p, seed, call=0, step=0, residual=None):
    """x with each element dropped (0, whatever it was) with probability p and the others scaled by 1 / (1 - p), plus `residual` (of x's
    shape and type) if there is one. p is rounded to a multiple of 2^-16, and the scale is that of the rounded one.

    The generator's key is the low 64 bits of `seed`, its counter the element's place in x (as if it were contiguous), `call`, which tells the dropouts of a step apart, and
    `step`: a number below 2^32, or one int32 or int64 on x's device, of which the kernel reads the low 32 bits, for steps that are captured
    into a graph (a parameter's step count of AdamW, for instance). Differentiable in x and residual, once; the gradient of x is this
    function of the gradient, with the step that was used."""
    seed = (operator.index(seed) + (1 << 63)) % (1 << 64) - (1 << 63)  # (64 bits, as the extension takes them; numpy's whole numbers too)
    if not 0 <= call < 1 << 32 or not (torch.is_tensor(step) or 0 <= step < 1 << 32):
        raise ValueError(f"call and step: 32 bits expected, got {call} and {step}")
    if torch.is_tensor(p) and p.requires_grad and torch.is_grad_enabled():
        raise ValueError("p: it gets no gradient")
    if forward_ad._current_level >= 0 or torch.jit.is_tracing() or _transformed(*(t for t in (x, residual, step, p) if torch.is_tensor(t))):
        return _Dropout.apply(x, p, seed, call, step, residual)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        ctx, stream = _where(x)
        number, at = (0, step) if torch.is_tensor(step) else (step, None)
        return _host().dropout_graph(ctx, stream, x, residual, p, seed, call, number, at)
    return _run(x.detach(), p, seed, call, step, None if residual is None else residual.detach(), False)[0]
