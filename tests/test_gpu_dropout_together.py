"""Dropout among other work: two streams at once, saved-tensor hooks, recomputed segments, a backward pass on a thread of its own."""
import threading

import pytest
import torch

from trips_amd.dropout import dropout

pytestmark = pytest.mark.gpu
SEED = 0x0123_4567_89AB_CDEF


def _pass(x, up, call, step, residual=None):
    out = dropout(x, 0.3, SEED, call=call, step=step, residual=residual)
    return out.detach(), *torch.autograd.grad(out, (x,) if residual is None else (x, residual), up)


def _sets(dtype):
    g = torch.Generator(device="cuda").manual_seed(6)
    return [(torch.randn(n, device="cuda", generator=g).to(dtype).requires_grad_(), torch.randn(n, device="cuda", generator=g).to(dtype), call) for n, call in ((3_000_001, 4), (999, 5))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams_at_once(dtype):
    """Each with its own tensors and its own step on the device, which goes on while the other runs."""
    sets, streams = _sets(dtype), [torch.cuda.Stream() for _ in range(2)]
    want = [[_pass(x, up, call, s) for s in range(1, 5)] for x, up, call in sets]
    steps = [torch.zeros((), dtype=torch.int32, device="cuda") for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                steps[i].add_(1)
                got[i].append(_pass(*sets[i], steps[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for one, other in zip(got, want) for p, q in zip(one, other) for a, b in zip(p, q))


@pytest.mark.parametrize("device_step", [True, False])
@pytest.mark.parametrize("with_residual", [True, False])
def test_saved_tensors_elsewhere(device_step, with_residual):
    """Hooks that move what is saved to the host and back; the step goes on in between."""
    (x, up, call), _ = _sets(torch.float32)
    r = torch.randn_like(x).requires_grad_() if with_residual else None
    want = _pass(x, up, call, 7, r)
    step = torch.full((), 7, dtype=torch.int64, device="cuda") if device_step else 7
    with torch.autograd.graph.save_on_cpu():
        out = dropout(x, 0.3, SEED, call=call, step=step, residual=r)
    if device_step:
        step.add_(1)
    got = (out.detach(), *torch.autograd.grad(out, (x, r) if with_residual else (x,), up))
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_hooks_that_pack_to_nothing_else():
    """What is saved of a step on the device is one number, and nothing of x."""
    (x, up, call), _ = _sets(torch.float32)
    sizes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (sizes.append(t.numel()), t)[1], lambda t: t):
        out = dropout(x, 0.3, SEED, call=call, step=torch.ones((), dtype=torch.int32, device="cuda"))
        dropout(x, 0.3, SEED, call=call, step=1)
    assert sizes == [1]
    assert torch.equal(torch.autograd.grad(out, x, up)[0], _pass(x, up, call, 1)[1])


def test_recomputed_segments():
    """The forward pass made again for the gradient drops the same elements."""
    from torch.utils.checkpoint import checkpoint
    (x, up, call), _ = _sets(torch.float32)
    step = torch.full((), 3, dtype=torch.int32, device="cuda")
    out = checkpoint(lambda a: torch.sin(dropout(torch.exp(a), 0.3, SEED, call=call, step=step)), x, use_reentrant=False)
    want = torch.sin(dropout(torch.exp(x), 0.3, SEED, call=call, step=3))
    assert torch.equal(out, want)
    assert torch.equal(torch.autograd.grad(out, x, up)[0], torch.autograd.grad(want, x, up)[0])


def test_a_backward_pass_on_another_thread():
    (x, up, call), _ = _sets(torch.bfloat16)
    want = _pass(x, up, call, 9)[1]
    out, got = dropout(x, 0.3, SEED, call=call, step=9), []
    thread = threading.Thread(target=lambda: got.append(torch.autograd.grad(out, x, up)[0]))
    thread.start(), thread.join(60)
    assert len(got) == 1 and torch.equal(got[0], want)
