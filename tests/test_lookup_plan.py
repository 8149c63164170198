"""What a LookupPlan keeps, on the CPU; what the kernels would return is stood in for."""
import pytest
import torch

from tests.test_lookup_modes import _Host
from trips_amd import lookup as lk


@pytest.fixture(autouse=True)
def host(monkeypatch):
    monkeypatch.setattr(lk, "_host", lambda: _Host)


def test_a_plans_own_index_is_kept_only_where_the_program_made_it():
    """A tensor that a render makes on the way (in a capture, on its own stream) is no one else's."""
    index = torch.tensor([2, 0, -1, 3], dtype=torch.int32)
    plan = lk.LookupPlan(torch.tensor([1, 0, 3, 2], dtype=torch.int32), torch.tensor([0, 1, 1, 2, 3], dtype=torch.int32), index)
    first, second = plan.own_index(index), plan.own_index(index)
    assert first.tolist() == second.tolist() == [0, 1, -1, 3]
    assert first.data_ptr() != second.data_ptr()
    plan.keep_own_index()
    kept = plan.own_index(index)
    assert kept.tolist() == [0, 1, -1, 3] and plan.own_index(index) is kept
    index[1] = 2
    with pytest.raises(ValueError, match="changed"):
        plan.own_index(index)


def test_plan_texels_keeps_it():
    from trips_amd.renderer import NeuralScene
    scene = NeuralScene(texture=torch.zeros(2, 4), background_color=torch.zeros(2), confidence=torch.zeros(1, 4), position=torch.zeros(4, 4),
                        point_size=torch.zeros(4, 1), index=torch.tensor([[2], [0], [2], [3]], dtype=torch.int32),
                        poses_se3=torch.zeros(1, 7, dtype=torch.float64), intrinsics=torch.zeros(1, 13))
    scene.plan_texels()
    index = scene.point_cloud_cuda.t_index
    assert scene.texel_plan.own_index(index) is scene.texel_plan.own_index(index)
    assert scene.texel_plan.own_index(index).tolist() == [[0], [1], [2], [3]]


def test_gradients_with_a_kept_plan_under_saved_tensor_hooks():
    """Hooks that hand back another tensor than the one that was saved (kept on the host, packed to disk)."""
    index = torch.tensor([2, 0, 2, 3], dtype=torch.int32)
    plan = lk.lookup_plan(index, 4)
    table = torch.randn(4, 3, requires_grad=True)
    want = torch.autograd.grad(lk.lookup(table, index, 2.0, lk.ROWS, plan).sum(), table)[0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.numpy().copy() if not t.requires_grad else t, lambda a: torch.from_numpy(a)):
        out = lk.lookup(table, index, 2.0, lk.ROWS, plan)
    assert torch.equal(torch.autograd.grad(out.sum(), table)[0], want)


def test_gradients_with_a_plan_that_was_written_to_are_refused():
    index = torch.tensor([2, 0, 2, 3], dtype=torch.int32)
    table = torch.randn(4, 3, requires_grad=True)
    for change in (lambda plan: plan.order.add_(0), lambda plan: plan.starts.add_(0), lambda plan: index.add_(0)):
        plan = lk.lookup_plan(index, 4)
        out = lk.lookup(table, index, 2.0, lk.ROWS, plan)
        change(plan)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_parameters_of_a_programs_own_kind_need_no_new_field(monkeypatch):
    """Any object with the fields that the render reads is taken as its parameters, also one without shared_texels_in_order."""
    from types import SimpleNamespace
    from trips_amd import renderer
    scene = renderer.NeuralScene(texture=torch.zeros(2, 4), background_color=torch.zeros(2), confidence=torch.zeros(1, 4), position=torch.zeros(4, 4),
                                 point_size=torch.zeros(4, 1), index=torch.zeros(4, 1, dtype=torch.int32),
                                 poses_se3=torch.zeros(1, 7, dtype=torch.float64), intrinsics=torch.zeros(1, 13))
    params = SimpleNamespace(add_depth_to_network=False, output_background_mask=False)
    info = renderer.NeuralRenderInfo(scene=scene, params=params)
    image = torch.zeros(1, 2, 3, 4)
    monkeypatch.setattr(renderer.PointRender, "render", staticmethod(lambda *a: ([image], None, None, None)))
    assert renderer.BlendPointCloud(info)[0] is image


def test_copies_of_a_plan_go_with_copies_of_their_index():
    """A scene that is copied or saved with its plan: the copy's index is what the plan was made of, whatever its version is."""
    import copy
    import pickle
    for changes in (0, 3):
        index = torch.tensor([2, 0, 2, 3], dtype=torch.int32)
        for _ in range(changes):
            index.add_(0)
        plan = lk.lookup_plan(index, 4)
        plan.keep_own_index()
        for twin, own in (copy.deepcopy((plan, index)), pickle.loads(pickle.dumps((plan, index))), (copy.copy(plan), index)):
            twin.check(own, 4)
            assert twin.own_index(own).tolist() == [0, 1, 2, 3] and torch.equal(twin.order, plan.order)
            if own is not index:
                with pytest.raises(ValueError, match="another index"):
                    twin.check(index, 4)
        index.add_(0)
        for twin, own in (copy.deepcopy((plan, index)), pickle.loads(pickle.dumps((plan, index))), (copy.copy(plan), index)):
            with pytest.raises(ValueError, match="changed"):  # (the index was written to since: so it is of a copy made now)
                twin.check(own, 4)


def test_a_plan_without_an_index_keeps_none():
    index = torch.tensor([2, 0, 2, 3], dtype=torch.int32)
    of = lk.lookup_plan(index, 4)
    plan = lk.LookupPlan(of.order, of.starts)
    with pytest.raises(ValueError, match="index"):
        plan.keep_own_index()
    assert plan.own_index(index).tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("confidence", [torch.zeros(1, 4, device="meta"), torch.zeros(1, 3), torch.zeros(1, 4, dtype=torch.float16)])
def test_what_the_splat_does_not_check_is_left_to_the_lookup(confidence, monkeypatch):
    """Without gradients too: another device's tensor, one shorter than the texture, one of another type."""
    from trips_amd import renderer
    scene = renderer.NeuralScene(texture=torch.zeros(2, 4), background_color=torch.zeros(2), confidence=confidence,
                                 position=torch.zeros(4, 4), point_size=torch.zeros(4, 1), index=torch.zeros(4, 1, dtype=torch.int32),
                                 poses_se3=torch.zeros(1, 7, dtype=torch.float64), intrinsics=torch.zeros(1, 13))
    info = renderer.NeuralRenderInfo(scene=scene, params=renderer.RenderParams(shared_texels_in_order=True), train=False)

    def lookup(*a, **kw):
        raise ValueError("looked up")
    monkeypatch.setattr(lk, "lookup", lookup)
    with pytest.raises(ValueError, match="looked up"):
        renderer.BlendPointCloud(info)


def test_a_plan_of_other_elements_at_the_same_address_is_refused():
    base = torch.tensor([0, 1, 2, 3, 0, 1, 2, 3, 0, 1, 2, 3], dtype=torch.int32)
    index, other = base.as_strided((4, 2), (3, 1)), base.as_strided((2, 4), (3, 1))
    plan = lk.LookupPlan(torch.arange(8, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), index)
    plan.check(base.as_strided((4, 2), (3, 1)), 4)
    with pytest.raises(ValueError, match="another index"):
        plan.check(other, 4)
