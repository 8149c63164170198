"""What AdamW keeps besides its kernels, on the CPU: its fields over load_state_dict, copies and refusals before a step."""
import pytest
import torch

from trips_amd.adamw import AdamW


def _optimiser(n=300, **kw):
    """An optimiser with the state that a first step would have made."""
    p = torch.nn.Parameter(torch.ones(n))
    opt = AdamW([p], **kw)
    opt.state[p] = dict(step=torch.ones((), dtype=torch.int32), first_moment=torch.full((n,), 0.25), second_moment=torch.full((n,), 0.5))
    return opt, p


def test_load_state_dict_keeps_copies_and_workspaces():
    opt, p = _optimiser()
    copy = torch.zeros(300, dtype=torch.bfloat16)
    opt.set_copy(p, copy)
    workspace, older, norm = torch.zeros(8), torch.zeros(4), torch.zeros(2)
    opt._workspace, opt._workspace_for, opt._norm, opt.grad_norm = workspace, 1, norm, norm
    opt._kept.append((older, norm))
    opt.load_state_dict(opt.state_dict())
    assert opt._copies[p] is copy
    assert opt._workspace is workspace and opt._norm is norm and opt.grad_norm is norm
    assert any(older is t for kept in opt._kept for t in kept)


def test_a_copied_optimiser_has_a_workspace_of_its_own():
    import copy
    import pickle
    opt, p = _optimiser(max_grad_norm=0.5, seed=3)
    opt.set_copy(p, torch.zeros(300))
    opt._workspace, opt._workspace_for, opt._norm, opt.grad_norm = torch.zeros(8), 1, torch.zeros(2), torch.zeros(2)
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert twin._workspace is None and twin.grad_norm is None and twin._kept == [] and twin._copies == {}
        assert (twin.max_grad_norm, twin.seed) == (0.5, 3)
        q = twin.param_groups[0]["params"][0]
        assert q is not p and torch.equal(twin.state[q]["first_moment"], opt.state[p]["first_moment"])


def test_state_bits_of_a_group_are_checked():
    p, q = torch.nn.Parameter(torch.ones(8)), torch.nn.Parameter(torch.ones(8))
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([dict(params=[p], state_bits=16)])
    opt = AdamW([dict(params=[p], state_bits=8)])
    with pytest.raises(ValueError, match="state_bits"):
        opt.add_param_group(dict(params=[q], state_bits=4))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[q]))
    assert [g["state_bits"] for g in opt.param_groups] == [8, 32]
    opt.param_groups[1]["state_bits"] = 16  # (set behind the optimiser's back: the first step makes no state)
    with pytest.raises(ValueError, match="state_bits"):
        opt._make_state(q, opt.param_groups[1])
    assert not opt.state.get(q)


def test_a_parameter_twice_in_a_group_is_refused():
    """Its two steps would run side by side in one launch, on the same weights and the same count."""
    p, q = torch.nn.Parameter(torch.ones(8)), torch.nn.Parameter(torch.ones(8))
    for params in ([p, p], [dict(params=[q, p, q])], [("a", p), ("b", p)]):
        with pytest.raises(ValueError, match="twice"):
            AdamW(params)
    opt = AdamW([p])
    with pytest.raises(ValueError, match="twice"):
        opt.add_param_group(dict(params=iter([q, q])))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=(x for x in [q])))
    assert len(opt.param_groups[1]["params"]) == 1
    with pytest.raises(ValueError):
        AdamW([dict(params=[p]), dict(params=[p])])  # (the base class)


def test_load_state_dict_goes_by_its_hooks():
    """Pre-hooks hand on another dict, post-hooks see the state loaded and may change it; later hooks come behind earlier ones."""
    opt, p = _optimiser()
    seen = []

    def first(o, sd):
        return {**sd, "state": {0: {**sd["state"][0], "step": torch.full((), 4, dtype=torch.int32)}}}

    def second(o, sd):
        seen.append(int(sd["state"][0]["step"]))
        return {**sd, "state": {0: {**sd["state"][0], "step": torch.full((), 5, dtype=torch.int32)}}}

    def after(o):
        seen.append(int(o.state[p]["step"]))
        o.state[p]["first_moment"].fill_(7.0)

    opt.register_load_state_dict_pre_hook(first), opt.register_load_state_dict_pre_hook(second)
    opt.register_load_state_dict_post_hook(after)
    saved = opt.state_dict()
    for _ in range(2):
        opt.load_state_dict(saved)
    assert seen == [4, 5, 4, 5] and int(opt.state[p]["step"]) == 5
    assert (opt.state[p]["first_moment"] == 7).all() and (saved["state"][0]["first_moment"] == 0.25).all()


def test_load_state_dict_keeps_types_and_what_is_no_parameters():
    p = torch.nn.Parameter(torch.ones(300, dtype=torch.bfloat16))
    opt = AdamW([p])
    opt.state[p] = dict(step=torch.ones((), dtype=torch.int32), first_moment=torch.ones(300).to(torch.float8_e4m3fn),
                        second_moment=torch.ones(300).to(torch.float8_e5m2), first_scale=torch.ones(2), second_scale=torch.ones(2))
    saved = opt.state_dict()
    saved["state"]["note"] = "kept"
    strided = dict(saved["state"][0], first_scale=torch.stack([torch.ones(2), torch.zeros(2)], 1)[:, 0])
    opt.load_state_dict(dict(saved, state={0: strided, "note": "kept"}))
    assert opt.state["note"] == "kept"
    for k, v in saved["state"][0].items():
        got = opt.state[p][k]
        assert got.dtype == v.dtype and got.is_contiguous() and got.data_ptr() != v.data_ptr() and torch.equal(got.float(), v.float())


def test_a_state_dict_that_does_not_fit_leaves_the_optimiser_alone():
    opt, p = _optimiser()
    saved = opt.state_dict()
    saved["param_groups"][0]["params"] = [0, 1]
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    assert (opt.state[p]["first_moment"] == 0.25).all() and len(opt._optimizer_load_state_dict_pre_hooks) == 0


def test_the_optimisers_own_options_are_in_its_state_dict():
    """A resumed run rounds with the same seed, and clips and scales as before, whatever it was made with."""
    opt, p = _optimiser(seed=11, max_grad_norm=0.5, skip_nonfinite=True)
    opt.loss_scale = 512.0
    saved = opt.state_dict()
    other, _ = _optimiser()
    other.load_state_dict(saved)
    assert (other.seed, other.max_grad_norm, other.skip_nonfinite, other.loss_scale) == (11, 0.5, True, 512.0)
    del saved["options"]  # (of a program that kept the rest alone)
    other, _ = _optimiser(seed=3)
    other.load_state_dict(saved)
    assert (other.seed, other.loss_scale) == (3, 1.0) and torch.equal(other.state[other.param_groups[0]["params"][0]]["first_moment"], torch.full((300,), 0.25))
