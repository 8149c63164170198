"""Lookups as programs use them: in front of the splat, under modes that torch has to see, with plans that are kept."""
import numpy as np
import pytest
import torch

from tests.test_gpu_operator import _info
from tests.test_gpu_shared_texels import _scene
from trips_amd import lookup as lk

pytestmark = pytest.mark.gpu


def _shared(seed, kept=False, **kw):
    from trips_amd.renderer import NeuralScene
    sc = _scene(seed, n=600)
    ns = NeuralScene.from_arrays(sc)
    if kept:
        ns.plan_texels()
    return ns, _info(sc, ns, shared_texels_in_order=True, **kw)


def _render_of(ns, info):
    from trips_amd.renderer import BlendPointCloud

    def render(t):
        ns.texture.texture = t
        return tuple(BlendPointCloud(info))
    return render


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("train", [False, True])
def test_forward_mode_of_shared_texels_is_refused(train, kept):
    import torch.autograd.forward_ad as fwad
    from trips_amd.renderer import BlendPointCloud
    ns, info = _shared(61, kept, train=train)
    plain = ns.texture.texture
    with torch.no_grad(), fwad.dual_level():
        ns.texture.texture = fwad.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(NotImplementedError):
            BlendPointCloud(info)
        ns.texture.texture = plain
        confidence = ns.texture.confidence_value_of_point
        ns.texture.confidence_value_of_point = fwad.make_dual(confidence, torch.ones_like(confidence))
        with pytest.raises(NotImplementedError):
            BlendPointCloud(info)


@pytest.mark.parametrize("transform", ["vmap", "grad", "jvp", "functionalize"])
def test_functional_transforms_of_shared_texels_are_refused(transform):
    ns, info = _shared(62, train=False)
    render, texture, f = _render_of(ns, info), ns.texture.texture.detach(), torch.func
    call = dict(vmap=lambda: f.vmap(render)(texture[None]), grad=lambda: f.grad(lambda t: render(t)[0].sum())(texture),
                jvp=lambda: f.jvp(render, (texture,), (texture,)), functionalize=lambda: f.functionalize(render)(texture))[transform]
    with torch.no_grad(), pytest.raises(RuntimeError):
        call()


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("train", [False, True])
def test_a_trace_of_shared_texels_renders_what_it_is_given(train, kept):
    ns, info = _shared(63, kept, train=train)
    render, texture = _render_of(ns, info), ns.texture.texture.detach().clone()
    with torch.no_grad():
        traced = torch.jit.trace(render, (texture,), check_trace=False)
        want, got = render(2 * texture), traced(2 * texture)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and float(want[0].abs().max()) > 0


def test_lookups_without_a_graph_under_modes():
    import torch.autograd.forward_ad as fwad
    index = torch.tensor([2, 0, -1, 3], dtype=torch.int32, device="cuda")
    table = torch.randn(4, 3, device="cuda")
    look = lambda t: lk.lookup(t, index, 2.0, lk.ROWS)
    with torch.no_grad():
        traced = torch.jit.trace(look, (table,), check_trace=False)
        assert torch.equal(traced(3 * table), look(3 * table))
        with fwad.dual_level(), pytest.raises(NotImplementedError):
            look(fwad.make_dual(table, table))
        with pytest.raises(RuntimeError):
            torch.func.vmap(look)(table[None])
        assert torch.equal(torch.func.vmap(lambda x: x + look(table).sum())(torch.zeros(2, device="cuda")), look(table).sum().expand(2))


@pytest.mark.parametrize("by_scene", [True, False])
def test_a_render_between_a_capture_and_its_first_replay(by_scene):
    """The first render with a plan is captured; an eager one before the replay, and the replays, give the same images. (With gradients
    asked for: without, the texels are not looked up.)"""
    from trips_amd.renderer import BlendPointCloud, NeuralScene
    sc = _scene(64, n=600)
    ns = NeuralScene.from_arrays(sc)
    ns.texture.texture.requires_grad_()
    with torch.enable_grad():
        want = [o.detach().clone() for o in BlendPointCloud(_info(sc, ns, train=False, shared_texels_in_order=True))]
        if by_scene:
            ns.plan_texels()
        else:
            ns.texel_plan = lk.lookup_plan(ns.point_cloud_cuda.t_index, ns.texture.texture.shape[1])
        captured, eager = (_info(sc, ns, train=False, shared_texels_in_order=True) for _ in range(2))
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            got = BlendPointCloud(captured)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(BlendPointCloud(eager), want))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("layout", [lk.COLUMNS, lk.ROWS])
def test_gradients_with_a_kept_plan_under_save_on_cpu(layout):
    rng = np.random.default_rng(7)
    index = torch.as_tensor(rng.integers(-1, 50, 3000), dtype=torch.int32, device="cuda")
    table = torch.randn((4, 50) if layout == lk.COLUMNS else (50, 4), device="cuda", requires_grad=True)
    weights = torch.randn((4, 3000) if layout == lk.COLUMNS else (3000, 4), device="cuda")
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            plan = lk.lookup_plan(index, 50)
        want = torch.autograd.grad((lk.lookup(table, index, 2.0, layout) * weights).sum(), table)[0]
        with torch.autograd.graph.save_on_cpu():
            out = lk.lookup(table, index, 2.0, layout, plan)
        assert torch.equal(torch.autograd.grad((out * weights).sum(), table)[0], want)
        checkpointed = torch.utils.checkpoint.checkpoint(lambda t: lk.lookup(t, index, 2.0, layout, plan), table, use_reentrant=False)
        assert torch.equal(torch.autograd.grad((checkpointed * weights).sum(), table)[0], want)


def test_hooks_that_hand_back_something_else_are_refused():
    index = torch.zeros(8, dtype=torch.int32, device="cuda")
    table = torch.ones(4, 5, device="cuda", requires_grad=True)
    plan = lk.lookup_plan(index, 5)
    for back in (lambda t: t.cpu(), lambda t: t.long() if t is not index else t, lambda t: t[:-1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            out = lk.lookup(table, index, 1.0, lk.COLUMNS, plan)
        with pytest.raises((ValueError, RuntimeError)):
            out.sum().backward()


def test_the_order_of_points_of_the_largest_table():
    texels = (1 << 31) - 2
    index = torch.tensor([texels - 1, 5, 0, texels, 1 << 30, 5, -1], dtype=torch.int64, device="cuda")
    plan = lk.lookup_plan(index, texels)
    assert plan.order.tolist() == [2, 1, 5, 4, 0, 3, 6]
    for first, behind, points in ((0, 1, 0), (1, 6, 1), (6, (1 << 30) + 1, 3), ((1 << 30) + 1, texels, 4), (texels, texels + 1, 5)):
        part = plan.starts[first:behind]
        assert part.numel() == behind - first and int(part.min()) == int(part.max()) == points


def test_a_copied_scene_renders_with_its_plan():
    import copy
    from trips_amd.renderer import BlendPointCloud
    ns, info = _shared(65, kept=True)
    twin = copy.deepcopy(ns)
    other = copy.copy(info)
    other.scene, other.cache = twin, None
    assert all(torch.equal(a, b) for a, b in zip(BlendPointCloud(info), BlendPointCloud(other)))
    twin.point_cloud_cuda.t_index[0] = 5
    with pytest.raises(ValueError, match="changed"):
        BlendPointCloud(other)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("kept", [False, True])
def test_a_frame_without_gradients_takes_no_lookups(kept, train, monkeypatch):
    """The splat reads shared texels by itself: the same images, nothing looked up, ordered or numbered on the way."""
    from trips_amd import renderer
    ns, info = _shared(66, kept, train=train)
    ns.texture.texture.requires_grad_()
    want = [o.detach() for o in renderer.BlendPointCloud(info)]

    def refuse(*a, **kw):
        raise AssertionError("a frame needs none of these")
    for name in ("lookup", "lookup_plan", "own_index"):
        monkeypatch.setattr(lk, name, refuse)
    with torch.no_grad():
        got = renderer.BlendPointCloud(info)
    ns.texture.texture.requires_grad_(False)
    again = renderer.BlendPointCloud(info)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, again))


@pytest.mark.parametrize("grad", [False, True])
def test_shared_texels_by_indexes_of_64_bits(grad):
    from trips_amd.renderer import BlendPointCloud
    ns, info = _shared(67)
    ns.texture.texture.requires_grad_(grad)
    want = BlendPointCloud(info)
    ns.point_cloud_cuda.t_index = ns.point_cloud_cuda.t_index.long()
    assert all(torch.equal(a, b) for a, b in zip(BlendPointCloud(info), want))
