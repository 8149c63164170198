"""The table's cross entropy and dropout where a mode is on that would lose what they compute, as lookups are tested: forward-mode
derivatives, functional transforms, traces. On the CPU; what the kernels would return is stood in for."""
import pytest
import torch

from trips_amd import dropout as dp
from trips_amd import table_loss as tl


class _Host:
    """The extension's calls, by detached torch operations: as little seen by torch as the kernels are."""

    @staticmethod
    def table_loss(ctx, stream, rows, table, target, scale, reduction):
        with torch.no_grad():
            return torch.nn.functional.cross_entropy(scale * rows @ table.t(), target.long(), reduction=("none", "sum", "mean")[reduction]), torch.cat([rows, target[:, None].float()], 1)

    @staticmethod
    def table_loss_backward(ctx, stream, grad, table, kept, n, scale, reduction, want_rows, want_table):
        with torch.enable_grad():
            x, w = kept[:, :-1].clone().requires_grad_(), table.clone().requires_grad_()
            loss = torch.nn.functional.cross_entropy(scale * x @ w.t(), kept[:, -1].long(), reduction=("none", "sum", "mean")[reduction])
            return torch.autograd.grad(loss, (x, w), grad)

    @staticmethod
    def dropout(ctx, stream, x, p, seed, call, step, step_at, residual, want_step):
        keep = torch.arange(x.numel()).reshape(x.shape) % 2 == 0
        out = torch.where(keep, x.detach() * 2, torch.zeros(()))
        return (out if residual is None else out + residual.detach()), (step_at.clone() if want_step and step_at is not None else None)


@pytest.fixture
def calls(monkeypatch):
    monkeypatch.setattr(tl, "_host", lambda: _Host)
    monkeypatch.setattr(dp, "_host", lambda: _Host)
    target = torch.tensor([2, 0, 3])
    table = torch.randn(4, 5)
    return {"loss": lambda t: tl.table_cross_entropy(t, table, target), "dropout": lambda t: dp.dropout(t, 0.5, 1)}


@pytest.mark.parametrize("which", ["loss", "dropout"])
@pytest.mark.parametrize("graph", [True, False])
def test_forward_mode_is_refused(calls, which, graph):
    import torch.autograd.forward_ad as fwad
    x = torch.randn(3, 5)
    with torch.set_grad_enabled(graph), fwad.dual_level():
        with pytest.raises(NotImplementedError):
            calls[which](fwad.make_dual(x, torch.ones_like(x)))
        calls[which](x)  # (no dual)


@pytest.mark.parametrize("which", ["loss", "dropout"])
@pytest.mark.parametrize("transform", ["vmap", "grad", "jvp", "functionalize"])
def test_functional_transforms_are_refused(calls, which, transform):
    f, x = calls[which], torch.randn(3, 5)
    call = dict(vmap=lambda: torch.func.vmap(f)(x[None]), grad=lambda: torch.func.grad(lambda t: f(t).sum())(x), jvp=lambda: torch.func.jvp(f, (x,), (x,)),
                functionalize=lambda: torch.func.functionalize(f)(x))[transform]
    with torch.no_grad(), pytest.raises(RuntimeError):
        call()


@pytest.mark.parametrize("which", ["loss", "dropout"])
@pytest.mark.parametrize("graph", [True, False])
def test_a_trace_records_the_call(calls, which, graph):
    f = calls[which]
    with torch.set_grad_enabled(graph):
        traced = torch.jit.trace(f, (torch.randn(3, 5),), check_trace=False)
        other = torch.randn(3, 5, requires_grad=graph)
        got = traced(other)
    with torch.no_grad():
        assert torch.equal(got, f(other))
    if graph:
        assert torch.autograd.grad(got.sum(), other)[0].shape == other.shape


def test_plain_tensors_under_a_transform_of_others(calls):
    x = torch.randn(3, 5)
    with torch.no_grad():
        for f in calls.values():
            got = torch.func.vmap(lambda a: a + f(x).sum())(torch.zeros(2))
            assert torch.equal(got, f(x).sum().expand(2))
