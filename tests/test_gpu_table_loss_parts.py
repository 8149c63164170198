"""Small problems of 16 bits hold d_ij in two parts: sums that are 0 show what one part would leave."""
import pytest
import torch

from tests import loss_parts
from trips_amd.table_loss import table_cross_entropy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,t,c", loss_parts.SIZES)
def test_two_parts(n, t, c, dtype):
    x, w, target, weights = loss_parts.zero_for_rows(n, t, c, dtype, "cuda")
    d = loss_parts.d(x, w, target, weights)
    x.requires_grad_(), w.requires_grad_()
    for reduction in ("none", "sum"):
        loss = table_cross_entropy(x, w, target, reduction=reduction)
        d_rows, = torch.autograd.grad(loss, x, torch.ones_like(loss))
        bound = loss_parts.bound(x.detach(), w.detach(), weights, d.abs().sum(1), t)
        assert (d_rows[:, 0].double().abs() <= bound).all(), float((d_rows[:, 0].double().abs() / bound).max())
    x, w, target, weights = loss_parts.zero_for_the_table(n, t, c, dtype, "cuda")
    sizes = loss_parts.d(x, w, target, weights).abs().t().contiguous() @ x.double().abs()
    w.requires_grad_()
    d_table, = torch.autograd.grad(table_cross_entropy(x, w, target, reduction="none"), w, weights)
    bound = loss_parts.bound(x, w.detach(), weights, sizes, x.shape[0])
    assert (d_table.double().abs() <= bound).all(), float((d_table.double().abs() / bound).max())
