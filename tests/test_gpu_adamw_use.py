"""AdamW as programs use it: resumed, captured, with copies that the forward reads, on other streams."""
import gc

import numpy as np
import pytest
import torch

from tests.test_gpu_adamw import TYPES, _check_step, _places, _state, _tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_and_captured_workspaces_after_load_state_dict(bits):
    """set_copy, then a checkpoint: later steps still write the copy; nor does what was captured lose its workspace."""
    from trips_amd.adamw import AdamW
    params, gs = _tensors((300, 5000), "f32", "f32", 21)
    given = dict(zip(params, gs))
    opt = AdamW(params, state_bits=bits, min_8bit_size=0, max_grad_norm=0.5)
    copies = [p.detach().to(torch.bfloat16) for p in params]
    for p, c in zip(params, copies):
        opt.set_copy(p, c)
    opt.step(grads=given)
    workspace, norm = opt._workspace.data_ptr(), opt.grad_norm.data_ptr()
    saved = opt.state_dict()
    opt.load_state_dict(saved)
    assert opt._workspace.data_ptr() == workspace and opt.grad_norm.data_ptr() == norm
    before = _state(opt, params)
    opt.step(grads=given)
    _check_step(opt, before, params, gs, 2, factor=float(opt.grad_norm[1]), places=_places(params))
    for p, c, w in zip(params, copies, before):
        assert torch.equal(c, p.detach().to(torch.bfloat16)) and not np.array_equal(p.detach().double().cpu().numpy(), w[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_backward_pass_that_needs_an_older_copy_raises(bits):
    """A step writes the copy: what autograd saved of it is gone, as with the parameter itself."""
    from trips_amd.adamw import AdamW
    params, gs = _tensors((300,), "f32", "f32", 22)
    opt = AdamW(params, state_bits=bits, min_8bit_size=0)
    copy = params[0].detach().to(torch.bfloat16)
    opt.set_copy(params[0], copy)
    opt.step(grads={params[0]: gs[0]})
    x = torch.ones(300, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    loss = (x * copy).sum()
    version = copy._version
    opt.step(grads={params[0]: gs[0]})
    assert copy._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        copy = params[0].detach().to(torch.float16)
    opt.set_copy(params[0], copy)
    opt.step(grads={params[0]: gs[0]})  # (has no version)
    assert torch.equal(copy, params[0].detach().to(torch.float16))


def test_a_backward_pass_that_needs_an_older_norm_raises():
    from trips_amd.adamw import AdamW
    params, gs = _tensors((300,), "f32", "f32", 23)
    opt = AdamW(params, max_grad_norm=0.5)
    opt.step(grads={params[0]: gs[0]})
    x = torch.ones(2, device="cuda", requires_grad=True)
    loss = (x * opt.grad_norm).sum()
    opt.step(grads={params[0]: gs[0]})
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_copies_that_changed_since_they_were_set_are_refused():
    from trips_amd.adamw import AdamW
    params, gs = _tensors((64,), "f32", "f32", 24)
    opt = AdamW(params)
    wide = torch.zeros(128, device="cuda")
    for other in (torch.zeros(64), wide[::2], torch.zeros(63, device="cuda"), torch.zeros(64, device="cuda", dtype=torch.float64)):
        copy = torch.zeros(64, device="cuda", dtype=other.dtype if other.dtype != torch.float64 else torch.float32)
        opt.set_copy(params[0], copy)
        if other.dtype == torch.float64:
            opt._copies[params[0]] = other
        else:
            copy.data = other
        before = params[0].detach().clone()
        with pytest.raises(RuntimeError, match="a copy"):
            opt.step(grads={params[0]: gs[0]})
        assert torch.equal(params[0], before) and not wide.any()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_steps_state_outlives_load_state_dict(bits):
    """What a graph writes is not given to others; it goes on with its own moments, and eager steps with those loaded."""
    from trips_amd.adamw import AdamW
    params, gs = _tensors((70_001, 9000), "f32", "f32", 25)
    given = dict(zip(params, gs))
    opt = AdamW(params, state_bits=bits, min_8bit_size=0, max_grad_norm=0.5)
    opt.step(grads=given)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        opt.step(grads=given)
    captured = {t.data_ptr() for p in params for t in opt.state[p].values()}
    import copy
    saved = copy.deepcopy(opt.state_dict())
    for _ in range(2):
        opt.load_state_dict(saved)
    others = [torch.zeros(n, dtype=d, device="cuda") for n in (70_001, 9000, 1, 274, 36) for d in (torch.float32, torch.uint8) for _ in range(20)]
    assert not captured & {t.data_ptr() for t in others + [t for p in params for t in opt.state[p].values()]}
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert not any(x.any() for x in others)
    assert all(int(opt.state[p]["step"]) == 1 for p in params)
    before = _state(opt, params)
    opt.step(grads=given)
    _check_step(opt, before, params, gs, 2, factor=float(opt.grad_norm[1]), places=_places(params))


def test_an_optimiser_dropped_while_its_step_runs_on_another_stream():
    """Its workspace, made on one stream, is not given to the next tensor of that stream while another one's step may write it."""
    from trips_amd.adamw import AdamW
    params, gs = _tensors((3000, 500), "f32", "f32", 26)
    opt = AdamW(params, max_grad_norm=0.5)
    opt.step(grads=dict(zip(params, gs)))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    kept = [(t.data_ptr(), t.data_ptr() + t.nbytes) for t in (opt._workspace, opt._norm)]
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)  # (some tenths of a second: the step waits behind it)
        opt.step(grads=dict(zip(params, gs)))
        done = side.record_event()
    del opt
    gc.collect()
    others = [torch.empty(16384, dtype=torch.uint8, device="cuda") for _ in range(300)]
    pending = not done.query()  # (a step that has ended by now shows nothing)
    torch.cuda.synchronize()
    inside = [t for t in others for a, b in kept if t.data_ptr() < b and a < t.data_ptr() + t.nbytes]
    assert not pending or not inside


@pytest.mark.parametrize("bits", [32, 8])
def test_workgroups_whose_tiles_belong_to_several_tensors(bits):
    """More than 2048 tiles, so that a workgroup has two, one behind the other; tensors that end after odd numbers of tiles. (Of a
    few million elements some moment (9 m + g) / 10 lies right on the border of two codes with most seeds; with this one none does.)"""
    from trips_amd.adamw import AdamW
    params, gs = _tensors((700_001, 2051, 1_000_077, 5, 400_000, 1, 1025), "f32", "f32", 32)
    opt = AdamW(params, state_bits=bits, min_8bit_size=0, seed=8)
    for t in (1, 2):
        before = _state(opt, params)
        opt.step(grads=dict(zip(params, gs)))
        _check_step(opt, before, params, gs, t, places=_places(params), seed=8)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_has_room_for(bits):
    from trips_amd.adamw import AdamW
    params, gs = _tensors([1 + i % 3 for i in range(4100)], "f32", "f32", 28)
    opt = AdamW(params, state_bits=bits, min_8bit_size=0, max_grad_norm=0.5, seed=9)
    before = _state(opt, params)
    opt.step(grads=dict(zip(params, gs)))
    _check_step(opt, before, params, gs, 1, factor=float(opt.grad_norm[1]), places=_places(params), seed=9)


@pytest.mark.parametrize("eps", [0.0, 1e-14])
@pytest.mark.parametrize("bits", [32, 8])
def test_an_eps_so_small_that_roots_are_taken_exactly(bits, eps):
    from trips_amd.adamw import AdamW
    params, gs = _tensors((1, 1027, 5000), "f32", "f32", 29)
    opt = AdamW(params, eps=eps, state_bits=bits, min_8bit_size=0, seed=10)
    for t in (1, 2):
        before = _state(opt, params)
        opt.step(grads=dict(zip(params, gs)))
        _check_step(opt, before, params, gs, t, places=_places(params), seed=10)
