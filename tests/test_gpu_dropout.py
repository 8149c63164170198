"""Dropout against numpy's Philox: an element is one product and one sum in float32, rounded once to its type."""
import numpy as np
import pytest
import torch

from tests.loss_reference import U, half_step, kept
from trips_amd.dropout import dropout

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SEED = 0xFEDC_BA98_7654_3210


def _numbers(t):
    return t.detach().double().cpu().numpy()


def _check(out, x, p, seed, call, step, residual=None):
    keep, factor = kept(x.numel(), p, seed, call, step)
    want = np.where(keep.reshape(x.shape), _numbers(x) * factor, 0.0)
    bound = 2 * U * np.abs(want)
    if residual is not None:
        want = want + _numbers(residual)
        bound = bound + U * np.abs(want)
    got = _numbers(out)
    assert got.shape == want.shape and out.dtype == x.dtype and out.is_contiguous()
    assert (np.abs(got - want) <= bound + half_step(x.dtype, want)).all()
    if residual is None:
        assert (got.reshape(-1)[~keep] == 0).all()
    return keep


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (2047,), (33, 31), (5, 3, 64), (1025, 1023), (3_000_001,)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_forward_and_gradients(dtype, shape, with_residual):
    g = torch.Generator(device="cuda").manual_seed(len(shape) + shape[0])
    x, r, up = (torch.randn(shape, device="cuda", generator=g).to(TYPES[dtype]) for _ in range(3))
    x.requires_grad_(), r.requires_grad_()
    out = dropout(x, 0.3, SEED, call=5, step=77, residual=r if with_residual else None)
    _check(out, x, 0.3, SEED, 5, 77, r if with_residual else None)
    with torch.no_grad():
        assert torch.equal(out, dropout(x, 0.3, SEED, 5, 77, r if with_residual else None))
    if with_residual:
        d_x, d_r = torch.autograd.grad(out, (x, r), up)
        assert torch.equal(d_r, up)
    else:
        d_x, = torch.autograd.grad(out, (x,), up)
    _check(d_x, up, 0.3, SEED, 5, 77)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -16, 0.1, 0.5, 0.99, 1.0 - 2.0 ** -16, 1.0 - 2.0 ** -18, 1.0])
def test_probabilities(p):
    x = torch.randn(100_001, device="cuda")
    keep = _check(dropout(x, p, 3), x, p, 3, 0, 0)
    # (within 6 deviations of its expectation; p rounded to 2^-16)
    q = np.round(p * 65536) / 65536
    assert abs(keep.mean() - (1 - q)) <= 6 * np.sqrt(q * (1 - q) / keep.size)


def test_dropped_elements_leave_nothing():
    x = torch.full((4096,), float("nan"), device="cuda")
    x[::2] = float("inf")
    keep, _ = kept(4096, 0.5, 9, 0, 0)
    got = dropout(x, 0.5, 9).cpu().numpy()
    assert (got[~keep] == 0).all() and not np.isfinite(got[keep]).any()
    assert (dropout(x, 1.0, 9) == 0).all()
    r = torch.randn(4096, device="cuda")
    assert torch.equal(dropout(x, 1.0, 9, residual=r), r)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_steps_on_the_device(index):
    """The step is read when the kernel runs; the gradient goes by the one that was used."""
    step = torch.full((), 41, dtype=index, device="cuda")
    x, up = torch.randn(1000, device="cuda", requires_grad=True), torch.randn(1000, device="cuda")
    out = dropout(x, 0.4, SEED, call=2, step=step)
    step.add_(1)
    d_x, = torch.autograd.grad(out, x, up)
    _check(out, x, 0.4, SEED, 2, 41)
    _check(d_x, up, 0.4, SEED, 2, 41)
    _check(dropout(x, 0.4, SEED, 2, step), x, 0.4, SEED, 2, 42)
    step.fill_(-1)
    _check(dropout(x, 0.4, SEED, 2, step), x, 0.4, SEED, 2, 0xFFFFFFFF)


def test_captured_steps_go_on():
    step = torch.zeros((), dtype=torch.int32, device="cuda")
    x, up = torch.randn(5000, device="cuda"), torch.randn(5000, device="cuda")

    def run():
        a = x.detach().requires_grad_()
        out = dropout(a, 0.25, SEED, 1, step)
        return out, torch.autograd.grad(out, a, up)[0]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step.add_(1)
        got = run()
    step.zero_()
    for i in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        assert int(step) == i
        _check(got[0], x, 0.25, SEED, 1, i)
        _check(got[1], up, 0.25, SEED, 1, i)
        assert all(torch.equal(a, b) for a, b in zip(run(), got))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_other_layouts(dtype):
    """An element's place is that of a contiguous x, whatever its strides; addresses of any element's alignment."""
    wide = torch.randn(40, 77, device="cuda").to(TYPES[dtype])
    for x in (wide.t(), wide[:, 1:70], wide[::3], wide.view(-1)[1:1000], wide.view(-1)[3:], wide[:1].expand(9, 77)):
        _check(dropout(x, 0.3, SEED), x, 0.3, SEED, 0, 0)
        _check(dropout(x, 0.3, SEED, residual=x), x, 0.3, SEED, 0, 0, x)
    assert dropout(wide[:0], 0.3, SEED).shape == (0, 77)


def test_far_elements():
    """Places beyond 2^32 (bfloat16, 8 GiB), against the oracle in a few windows."""
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    out = dropout(x, 0.5, SEED, 3, 4)
    for first in (0, 1 << 31, (1 << 32) - 4096, 1 << 32):
        size = min(4096, n - first)
        keep, factor = kept(size, 0.5, SEED, 3, 4, first)
        assert np.array_equal(out[first:first + size].float().cpu().numpy(), keep * factor)
    keep, _ = kept(3, 0.5, SEED, 3, 4, n - 3 - (n - 3) % 8)
    assert float(out[n - 3]) in (0.0, 2.0)


def test_gradients_once_and_refusals():
    x = torch.randn(64, device="cuda", requires_grad=True)
    d, = torch.autograd.grad(dropout(x, 0.5, 1).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), x)
    for kw, message in ((dict(p=1.5), "p:"), (dict(p=float("nan")), "p:"), (dict(p=-0.1), "p:"), (dict(call=-1), "32 bits"), (dict(call=1 << 32), "32 bits"), (dict(step=-1), "32 bits"),
                        (dict(step=torch.zeros(2, dtype=torch.int32, device="cuda")), "step"), (dict(step=torch.zeros((), device="cuda")), "step"),
                        (dict(step=torch.zeros((), dtype=torch.int32)), "step"), (dict(residual=torch.zeros(63, device="cuda")), "residual"),
                        (dict(residual=torch.zeros(64, device="cuda", dtype=torch.float16)), "residual")):
        with pytest.raises(ValueError, match=message):
            dropout(x, **{"p": 0.5, "seed": 1, **kw})
    with pytest.raises(ValueError, match="x:"):
        dropout(x.detach().double(), 0.5, 1)
    with pytest.raises(RuntimeError, match="GPU"):
        dropout(torch.zeros(4), 0.5, 1)
