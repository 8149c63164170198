"""A scale that something would be differentiated by: refused, since the cross entropy has no gradient for it. On the CPU, over test_loss_modes' stand-in."""
import pytest
import torch

from tests.test_loss_modes import _Host
from trips_amd import table_loss as tl


@pytest.fixture
def loss(monkeypatch):
    class Host(_Host):
        @staticmethod
        def table_loss(ctx, stream, rows, table, target, scale, reduction):  # (a number, as the extension takes it)
            return _Host.table_loss(ctx, stream, rows, table, target, float(scale), reduction)
    monkeypatch.setattr(tl, "_host", lambda: Host)
    rows, table, target = torch.randn(3, 5), torch.randn(4, 5), torch.tensor([2, 0, 3])
    return lambda scale: tl.table_cross_entropy(rows, table, target, scale=scale)


def test_a_scale_that_is_learned_is_refused(loss):
    scale = torch.tensor(0.5, requires_grad=True)
    with pytest.raises(ValueError, match="scale"):
        loss(scale)
    with torch.no_grad():
        assert torch.equal(loss(scale), loss(0.5))
    assert torch.equal(loss(scale.detach()), loss(0.5))


def test_a_dual_scale_is_refused(loss):
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        loss(fwad.make_dual(torch.tensor(0.5), torch.tensor(1.0)))


@pytest.mark.parametrize("transform", ["grad", "jvp", "vmap"])
def test_a_transformed_scale_is_refused(loss, transform):
    scale = torch.tensor(0.5)
    call = dict(grad=lambda: torch.func.grad(loss)(scale), jvp=lambda: torch.func.jvp(loss, (scale,), (scale,)), vmap=lambda: torch.func.vmap(loss)(scale[None]))[transform]
    with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
        call()
