"""Seeds as programs have them, and the 64 bits that the extension gets of them. On the CPU, over a stand-in."""
import numpy as np
import pytest
import torch

from trips_amd import dropout as dp


@pytest.mark.parametrize("seed,want", [(5, 5), (np.int64(5), 5), (np.int32(-2), -2), (np.uint64(2 ** 64 - 1), -1), (2 ** 63, -2 ** 63), (-2 ** 63, -2 ** 63), (2 ** 64 + 7, 7), (True, 1), (torch.tensor(9), 9)])
@pytest.mark.parametrize("grad", [False, True])
def test_seeds(monkeypatch, seed, want, grad):
    got = []

    class Host:
        @staticmethod
        def dropout(ctx, stream, x, p, seed, *rest):
            got.append(seed)
            return x, None

        @staticmethod
        def dropout_graph(ctx, stream, x, residual, p, seed, *rest):
            got.append(seed)
            return x
    monkeypatch.setattr(dp, "_host", lambda: Host)
    dp.dropout(torch.zeros(3, requires_grad=grad), 0.5, seed)
    assert got == [want] and type(got[0]) is int


@pytest.mark.parametrize("seed", [1.5, 1.0, "1", None, np.float64(2), torch.tensor(1.0)])
def test_seeds_that_are_no_whole_numbers(seed):
    with pytest.raises(TypeError):
        dp.dropout(torch.zeros(3), 0.5, seed)


def test_a_probability_that_something_is_differentiated_by_is_refused(monkeypatch):
    """Dropout has no gradient for it."""
    import torch.autograd.forward_ad as fwad

    class Host:
        @staticmethod
        def dropout(ctx, stream, x, p, *rest):
            return x * (1 / (1 - float(p))), None
    monkeypatch.setattr(dp, "_host", lambda: Host)
    x, p = torch.ones(3), torch.tensor(0.5, requires_grad=True)
    with pytest.raises(ValueError, match="p:"):
        dp.dropout(x, p, 1)
    with torch.no_grad():
        assert torch.equal(dp.dropout(x, p, 1), x * 2)
    assert torch.equal(dp.dropout(x, p.detach(), 1), x * 2)
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        dp.dropout(x, fwad.make_dual(torch.tensor(0.5), torch.tensor(1.0)), 1)
    for call in (lambda: torch.func.grad(lambda q: dp.dropout(x, q, 1).sum())(p.detach()), lambda: torch.func.vmap(lambda q: dp.dropout(x, q, 1))(p.detach()[None])):
        with pytest.raises((RuntimeError, ValueError)):
            call()
