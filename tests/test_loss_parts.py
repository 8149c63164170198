"""What loss_parts holds two parts of d_ij to is beyond one part, and beyond a second part that is dropped for half of the rows, or taken twice. On the CPU: planted in the oracle."""
import pytest
import torch

from tests import loss_parts


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,t,c", loss_parts.SIZES)
@pytest.mark.parametrize("which", ["rows", "table"])
def test_one_part_is_outside_the_bound(n, t, c, which, dtype):
    x, w, target, weights = (loss_parts.zero_for_rows if which == "rows" else loss_parts.zero_for_the_table)(n, t, c, dtype)
    d = loss_parts.d(x, w, target, weights)
    held = 32768.0 / float(weights.abs().max()) if dtype is torch.float16 else 1.0
    one = (d * held).to(dtype).double() / held
    two = one + ((d - one) * held).to(dtype).double() / held
    if which == "rows":
        product, terms = (lambda a: (a @ w.double())[:, 0]), t
        sizes = d.abs().sum(1)
    else:
        product, terms = (lambda a: a.t() @ x.double()), x.shape[0]
        sizes = d.abs().t() @ x.double().abs()
    bound = loss_parts.bound(x, w, weights, sizes, terms)
    assert (product(d).abs() < bound / 64).all()
    assert (product(two).abs() <= bound).all()
    twice = 2 * two - one
    for wrong in (one, twice):
        outside = product(wrong).abs() > bound
        assert outside.any() and (n < 20 or outside.double().mean() > 0.1), float(outside.double().mean())
