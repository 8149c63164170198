"""A table's cross entropy over very many rows, which are taken in blocks, against loss_sums in double precision."""
import pytest
import torch

from tests import loss_sums
from tests.loss_sums import U
from trips_amd.table_loss import table_cross_entropy

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 1 << 20  # rows


def _within(got, want, bound, what):
    """(What is beyond the type's numbers is infinite: a million times one row's gradient in float16.)"""
    most, got = torch.finfo(got.dtype).max, got.double()
    off = torch.where((want.abs() + bound > most) & (want * got > most * want.abs()), 0.0, (got - want).abs())
    assert (off <= bound).all(), f"{what}: {float((off / bound).max()):.3g} times the bound"


def _check(n, t, c, padding, dtype, reduction="mean", scramble=None):
    x, w, target = loss_sums.inputs(n, t, c, padding, TYPES[dtype], "cuda")
    if scramble is not None:
        target = scramble(target)
    g = torch.Generator(device="cuda").manual_seed(3)
    up = torch.rand(n, device="cuda", generator=g) + 0.5 if reduction == "none" else torch.tensor(1.5 if reduction == "sum" else 1e6, device="cuda")
    count = max(1, int((target >= 0).sum()))
    weights = up if reduction == "none" else (up / (count if reduction == "mean" else 1)).expand(n)
    if dtype == "f16" and reduction != "mean":
        weights, up = weights / 4096, up / 4096  # (sums of a million rows are beyond its range)
    x.requires_grad_(), w.requires_grad_()
    loss = table_cross_entropy(x, w, target, reduction=reduction)
    d_rows, d_table = torch.autograd.grad(loss, (x, w), up)
    want_rows, rows_size, want, size = loss_sums.gradients(x, w, target, weights)
    bound = loss_sums.table_bound(x, w, n, want, size)
    low = 2.0 ** -24 * count * float(weights.max()) / 32768 * 1.25 if dtype == "f16" else 0.0  # (the smallest step of d_ij as float16 holds it)
    _within(d_table, want, bound + low, "d_table")
    step = torch.finfo(x.dtype).eps
    far = (step + (t + 2 * c + 32) * 4 * U) * rows_size + step / 2 * want_rows.abs() + 2.0 ** -24 * float(weights.max()) / 32768 * t + 2.0 ** -25
    _within(d_rows, want_rows, far, "d_rows")
    assert (d_rows[target < 0] == 0).all()
    return x, w, target, up, d_rows, d_table


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,t,c,padding,reduction", [(BLOCK, 40, 6, 0.0, "mean"), (BLOCK + 1, 40, 6, 0.0, "none"), (1_100_000, 40, 6, 0.3, "mean"), (2_300_000, 150, 16, 0.1, "sum"),
                                                     (3_000_001, 7, 3, 0.7, "none"), (1_500_000, 300, 17, 0.2, "mean"), (1_100_000, 1100, 40, 0.0, "mean")])
def test_many_rows(n, t, c, padding, reduction, dtype):
    _check(n, t, c, padding, dtype, reduction)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_rows_of_a_large_table(dtype):
    """Several pieces of the table and several blocks of the rows, in tiles of 128."""
    _check(1_060_000, 2060 if dtype == "f32" else 4097, 1024 if dtype == "bf16" else 260, 0.1, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("which", ["none", "one", "first block", "but one", "far apart"])
def test_blocks_without_rows_that_count(which, dtype):
    n = 2 * BLOCK + 77
    at = torch.arange(n, device="cuda")
    keep = {"none": at < 0, "one": at == n - 5, "first block": at < n // 3, "but one": at != 12, "far apart": at % 4099 == 5}[which]
    _check(n, 30, 5, 0.0, dtype, "mean", lambda target: torch.where(keep, target, -1))


def test_many_rows_captured_and_again():
    """The same bits every time, also from a graph, and from a workspace that held other numbers."""
    x, w, target, up, d_rows, d_table = _check(1_300_000, 90, 12, 0.2, "bf16")

    def step():
        return torch.autograd.grad(table_cross_entropy(x, w, target), (x, w), up)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    x, w = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        again = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, again, (d_rows, d_table)))


def test_one_gradient_of_many_rows():
    x, w, target, up, d_rows, d_table = _check(1_300_000, 90, 12, 0.2, "f32")
    assert torch.equal(torch.autograd.grad(table_cross_entropy(x, w.detach(), target), x, up)[0], d_rows)
    assert torch.equal(torch.autograd.grad(table_cross_entropy(x.detach(), w, target), w, up)[0], d_table)
