"""A table's cross entropy of widths, strides and shapes at the ends of what it takes; the bounds are loss_reference.Loss's."""
import numpy as np
import pytest
import torch

from tests.loss_reference import Loss, within
from trips_amd.table_loss import table_cross_entropy

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _inputs(n, t, c, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + n + 7 * t + 31 * c)
    x, w = torch.randn(n, c, device="cuda", generator=g), torch.randn(t, c, device="cuda", generator=g) * (2 / c ** 0.5)
    target = torch.randint(0, t, (n,), device="cuda", generator=g)
    target[::5] = -1
    return (x + w[target.clamp(min=0)]).to(TYPES[dtype]), w.to(TYPES[dtype]), target


def _check(x, w, target, scale=1.0):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    want = Loss(x, w, target, scale, (target.reshape(-1) >= 0).cpu().numpy().astype(np.float64))
    loss = table_cross_entropy(x, w, target, scale=scale, reduction="none")
    got = (loss.detach(), *torch.autograd.grad(loss.sum(), (x, w)))
    for a, b, bound, what in zip(got, (want.losses, want.d_rows, want.d_table), (want.loss_bound, want.d_rows_bound, want.d_table_bound), ("loss", "d_rows", "d_table")):
        within(a, b, bound, what)
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,t,c", [(1, 2, 131_071), (3, 5, 131_070), (40, 30, 70_001), (300, 20, 131_071), (200, 150, 40_000)])
def test_the_widest_rows(n, t, c, dtype):
    _check(*_inputs(n, t, c, dtype))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("stride", [(1 << 20) - 8, 1 << 20, (1 << 20) + 1])
def test_far_strides(dtype, stride):
    """Rows farther apart than the direct loads reach are copied."""
    x, w, target = _inputs(30, 70, 40, dtype)
    want = _check(x, w, target)
    far = [torch.empty(m.shape[0], stride, dtype=m.dtype, device="cuda")[:, :40].copy_(m) for m in (x, w)]
    assert far[1].stride() == (stride, 1)
    assert all(torch.equal(a, b) for a, b in zip(_check(*far, target), want))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("stride", [0, 1, 2, 6])
def test_rows_that_overlap(dtype, stride):
    """Entries that are windows of one row of memory, or all the same: read where they are, with what a copy of them gives."""
    for n, t, c in ((20, 300, 24), (300, 700, 33), (5, 4000, 10)):
        x, _, target = _inputs(n, t, c, dtype)
        memory = _inputs(1, 1, (t - 1) * stride + c, dtype)[0]
        windows = memory.as_strided((t, c), (stride, 1))
        x.requires_grad_()
        apart = windows.contiguous().requires_grad_()
        want = table_cross_entropy(x, apart, target)
        got = table_cross_entropy(x, windows, target)
        assert torch.equal(got, want)
        assert torch.equal(torch.autograd.grad(got, x)[0], torch.autograd.grad(want, x)[0])
    rows = memory.as_strided((300, 10), (min(stride, 2), 1))  # (and rows that do)
    w, target = _inputs(2, 50, 10, dtype)[1], torch.arange(300, device="cuda") % 50
    assert torch.equal(table_cross_entropy(rows, w, target), table_cross_entropy(rows.contiguous(), w, target))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_targets_of_any_shape(dtype):
    x, w, target = _inputs(120, 90, 32, dtype)
    want = _check(x, w, target)
    for shaped in (target.view(10, 12), target.view(2, 3, 20), target.view(12, 10).t().contiguous().t(), target.to(torch.int32).view(120, 1), torch.stack([target, target], 1)[:, 0]):
        assert all(torch.equal(a, b) for a, b in zip(_check(x, w, shaped), want))
    alone = table_cross_entropy(x[1:2], w, target[1])
    assert alone.shape == () and torch.equal(alone, table_cross_entropy(x[1:2], w, target[1:2]))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_a_texture_turned(dtype):
    """A table in the layout of a scene's texture, [C, T]."""
    x, w, target = _inputs(70, 400, 4, dtype)
    texture = w.t().contiguous().requires_grad_()
    want = _check(x, w, target)
    loss = table_cross_entropy(x, texture.t(), target, reduction="none")
    assert torch.equal(loss, want[0])
    d, = torch.autograd.grad(loss.sum(), texture)
    assert d.shape == texture.shape and torch.equal(d.t(), want[2])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_are_the_table(dtype):
    """Both gradients of one tensor, added up by torch."""
    _, w, _ = _inputs(1, 90, 24, dtype)
    w.requires_grad_()
    target = (torch.arange(90, device="cuda") + 1) % 90
    got, = torch.autograd.grad(table_cross_entropy(w, w, target), w)
    x, y = w.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    d = torch.autograd.grad(table_cross_entropy(x, y, target), (x, y))
    assert torch.equal(got, d[0] + d[1])
