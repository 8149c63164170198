"""Lookups without a graph where a mode is on that would lose what they compute: forward-mode derivatives, functional transforms,
traces. On the CPU; what the kernels would return is stood in for."""
import numpy as np
import pytest
import torch

from trips_amd import lookup as lk


class _Host:
    """The extension's calls (in rows), by numpy: as little seen by torch as the kernels are."""

    @staticmethod
    def lookup(ctx, stream, table, index, scale, layout):
        return torch.from_numpy(table.numpy()[index.numpy()] * np.float32(scale))

    @staticmethod
    def lookup_backward(ctx, stream, grad, index, order, starts, texels, scale, layout, out):
        got = np.zeros((texels, grad.shape[1]), np.float32)
        np.add.at(got, index.numpy(), grad.detach().numpy() * np.float32(scale))
        return torch.from_numpy(got)

    @staticmethod
    def lookup_plan(ctx, stream, index, texels):
        i = index.numpy().reshape(-1)
        return (torch.from_numpy(np.argsort(i, kind="stable").astype(np.int32)),
                torch.from_numpy(np.searchsorted(np.sort(i), np.arange(texels + 1)).astype(np.int32)))


@pytest.fixture
def rows(monkeypatch):
    monkeypatch.setattr(lk, "_host", lambda: _Host)
    index = torch.tensor([2, 0, 2, 3], dtype=torch.int32)
    return lambda t: lk.lookup(t, index, 2.0, lk.ROWS), index


@pytest.mark.parametrize("graph", [True, False])
def test_forward_mode_is_refused(rows, graph):
    import torch.autograd.forward_ad as fwad
    look, index = rows
    table = torch.randn(4, 3)
    with torch.set_grad_enabled(graph), fwad.dual_level():
        dual = fwad.make_dual(table, torch.ones_like(table))
        with pytest.raises(NotImplementedError):
            look(dual)
        with pytest.raises(NotImplementedError):
            lk.lookup_backward(dual, index, 4, layout=lk.ROWS)
        assert torch.equal(look(table), table[index.long()] * 2)  # (no dual)


def test_forward_mode_over_the_gradient_is_refused(rows):
    """A tangent of what comes back to the lookup."""
    import torch.autograd.forward_ad as fwad
    look, _ = rows
    table = torch.randn(4, 3, requires_grad=True)
    with fwad.dual_level():
        weights = fwad.make_dual(torch.ones(4, 3), torch.ones(4, 3))
        with pytest.raises(NotImplementedError):
            torch.autograd.grad((look(table) * weights).sum(), table)


@pytest.mark.parametrize("transform", ["vmap", "grad", "jvp", "functionalize"])
def test_functional_transforms_are_refused(rows, transform):
    look, index = rows
    table = torch.randn(4, 3)
    for f in (look, lambda t: lk.lookup_backward(t, index, 4, layout=lk.ROWS)):
        call = dict(vmap=lambda: torch.func.vmap(f)(table[None]), grad=lambda: torch.func.grad(lambda t: f(t).sum())(table),
                    jvp=lambda: torch.func.jvp(f, (table,), (table,)), functionalize=lambda: torch.func.functionalize(f)(table))[transform]
        with torch.no_grad(), pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("graph", [True, False])
def test_a_trace_looks_up_what_it_is_given(rows, graph):
    look, index = rows
    table = torch.randn(4, 3)
    with torch.set_grad_enabled(graph):
        traced = torch.jit.trace(look, (table,), check_trace=False)
        other = torch.randn(4, 3, requires_grad=graph)
        got = traced(other)
        assert torch.equal(got, other[index.long()] * 2)
    if graph:
        got.sum().backward()
        assert torch.equal(other.grad, torch.bincount(index.long(), minlength=4)[:, None].float().expand(4, 3) * 2)


def test_what_a_trace_would_not_record_is_refused(rows):
    _, index = rows
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda g: lk.lookup_backward(g, index, 4, layout=lk.ROWS), (torch.ones(4, 3),), check_trace=False)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda i: lk.lookup_plan(i, 4).order, (index,), check_trace=False)


def test_a_traced_lookup_refuses_the_plan_of_another_index(rows):
    _, index = rows
    table, plan = torch.randn(4, 3), lk.lookup_plan(index, 4)
    traced = torch.jit.trace(lambda t, i: lk.lookup(t, i, 1.0, lk.ROWS, plan), (table, index), check_trace=False)
    assert torch.equal(traced(2 * table, index), 2 * table[index.long()])
    with pytest.raises(RuntimeError, match="plan"):
        traced(table, index.clone())


def test_plain_tensors_under_a_transform_of_others(rows):
    """A table that the transform does not follow is looked up as ever."""
    look, index = rows
    table = torch.randn(4, 3)
    with torch.no_grad():
        got = torch.func.vmap(lambda x: x + look(table).sum())(torch.zeros(2))
        assert torch.equal(got, (table[index.long()] * 2).sum().expand(2))
