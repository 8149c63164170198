"""The bound of loss_sums on sums over very many rows sees a part of the rows that is left out. On the CPU: the mistakes are planted in the oracle."""
import pytest
import torch

from tests import loss_sums


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,t,c,padding", [(1_100_000, 40, 6, 0.3), (2_300_000, 6, 4, 0.0)])
def test_a_part_that_is_left_out_is_outside_the_bound(n, t, c, padding, dtype):
    x, w, target = loss_sums.inputs(n, t, c, padding, dtype, "cpu")
    weights = torch.ones(n)
    _, _, want, size = loss_sums.gradients(x, w, target, weights)
    bound = loss_sums.table_bound(x, w, n, want, size)
    assert (bound <= want.abs() / 100)[t // 2 + 1:].all()
    for parts, which in ((64, 0), (64, 17), (64, 63), (16, 5), (2, 1)):
        gone = torch.zeros(n, dtype=torch.bool)
        gone[n * which // parts:n * (which + 1) // parts] = True
        wrong = loss_sums.gradients(x, w, target, weights, gone)[2]  # (added twice it is as far off)
        assert ((wrong - want).abs() > bound)[t // 2 + 1:].all(), (parts, which)
    assert (torch.zeros_like(want) - want).abs().gt(bound).all()
