"""Points that share texels: the render operator with RenderParams.shared_texels_in_order, and a training step of the whole
chain as it would be used: shared descriptors looked up, splat, net, loss, gradients in order, norm, AdamW."""
import numpy as np
import pytest
import torch

from tests import optim_reference as ref
from tests.test_gpu_operator import _info
from trips_amd import abi, scenes

pytestmark = pytest.mark.gpu
TEXELS = 700


def _scene(seed, n=5000, outside=0, layers=4):
    """A scene whose points share TEXELS texels; a few with none."""
    sc = scenes.tiny(n=n, w=80, h=60, f=70.0, num_layers=layers, list_depth=16, seed=seed, views=2, radius=(0.004, 0.4))
    rng = np.random.default_rng(seed)
    sc.index = (TEXELS * rng.random(n) ** 2).astype(np.int32)
    sc.texture = np.ascontiguousarray(sc.texture[:, :TEXELS])
    sc.confidence = np.ascontiguousarray(np.asarray(sc.confidence).reshape(-1)[:TEXELS])
    if outside:
        sc.index[rng.permutation(n)[:outside]] = -1
    return sc


def _train(sc, in_order, kept=False, seed=0):
    from trips_amd.renderer import BlendPointCloud, NeuralScene
    ns = NeuralScene.from_arrays(sc, requires_grad=True)
    info = _info(sc, ns, shared_texels_in_order=in_order)
    if kept:
        ns.plan_texels()
    outs = BlendPointCloud(info)
    rng = np.random.default_rng(seed)
    grads = [rng.normal(0, 1, o.shape).astype(np.float32) for o in outs]
    sum((o * torch.as_tensor(g).cuda()).sum() for o, g in zip(outs, grads)).backward()
    return ns, outs, grads


def test_images_gradients_and_their_bits(oracle):
    from tests.gpu_util import assert_grad_close
    sc = _scene(51)
    ns, outs, grads = _train(sc, True)
    d = abi.desc_for_scene(sc)
    assert d.num_texels == TEXELS
    want = oracle.forward(sc, d)
    for a, b in zip(outs, want["images"]):
        np.testing.assert_allclose(a.detach().cpu().numpy(), b, rtol=1e-5, atol=1e-6)
    g = oracle.backward(sc, d, want, grads)
    for key, got in (("d_texture", ns.texture.texture.grad), ("d_background", ns.texture.background_color.grad),
                     ("d_position", ns.point_cloud_cuda.t_position.grad), ("d_pose", ns.poses.tangent_poses.grad),
                     ("d_intrinsics", ns.intrinsics.intrinsics.grad),
                     ("d_confidence", ns.texture.confidence_value_of_point.grad.reshape(-1)),
                     ("d_point_size", ns.point_cloud_cuda.t_point_size.grad.reshape(-1))):
        assert_grad_close(key, got.cpu().numpy(), g[key])
    assert ns.texture.confidence_value_of_point.grad.shape == (1, TEXELS)
    direct, images, _ = _train(sc, False)
    assert all(torch.equal(a, b) for a, b in zip(outs, images))
    assert torch.equal(direct.point_cloud_cuda.t_position.grad, ns.point_cloud_cuda.t_position.grad)
    for kept in (False, True):
        again, _, _ = _train(sc, True, kept)
        assert torch.equal(again.texture.texture.grad, ns.texture.texture.grad)
        assert torch.equal(again.texture.confidence_value_of_point.grad, ns.texture.confidence_value_of_point.grad)


def test_points_without_a_texel_are_left_out_and_reported():
    from trips_amd._lib import TripsError
    from trips_amd.renderer import BlendPointCloud, NeuralScene, get_context
    sc = _scene(52, outside=40)
    for train in (True, False):
        got = []
        for in_order in (False, True):
            ns = NeuralScene.from_arrays(sc)
            info = _info(sc, ns, train=train, shared_texels_in_order=in_order)
            got.append(BlendPointCloud(info))
            with pytest.raises(TripsError, match="outside"):
                get_context(0).check(info.cache.workspace)
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_a_plan_of_an_older_index_is_refused():
    from trips_amd.renderer import BlendPointCloud, NeuralScene
    sc = _scene(53)
    ns = NeuralScene.from_arrays(sc)
    ns.plan_texels()
    ns.point_cloud_cuda.t_index[0] = 5
    with pytest.raises(ValueError, match="plan"):
        BlendPointCloud(_info(sc, ns, shared_texels_in_order=True))


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_of_the_whole_chain(bits):
    """Three steps. Gradients of shared descriptors against indexing in torch around the same splat; the norm and every step of
    AdamW against the formulas in double; the shared texels' gradients of the first step with the same bits in a second run (not
    of later ones: the net's sums for its last layer's weights are not always in one order, and they step the net)."""
    from trips_amd.adamw import AdamW
    from trips_amd.renderer import BlendPointCloud, NeuralScene
    from trips_amd.unet import MultiScaleUnet2dDecOnlySmallFixed, MultiScaleUnet2dParams
    sc = _scene(54)
    runs, first = [], []
    for _ in range(2):
        ns = NeuralScene.from_arrays(sc)
        texture, confidence = torch.nn.Parameter(ns.texture.texture), torch.nn.Parameter(ns.texture.confidence_value_of_point)
        ns.texture.texture, ns.texture.confidence_value_of_point = texture, confidence
        ns.plan_texels()
        net = MultiScaleUnet2dDecOnlySmallFixed(MultiScaleUnet2dParams(num_input_layers=4, num_layers=4, filters_network=[16, 32, 32, 32]))
        net = net.he_normal_(torch.Generator().manual_seed(1)).cuda()
        params = [texture, confidence, *net.parameters()]
        opt = AdamW([dict(params=params[:2], lr=1e-3, weight_decay=0.0), dict(params=params[2:], lr=1e-4)], state_bits=bits,
                    min_8bit_size=256, max_grad_norm=0.05, seed=11)
        target = torch.rand((2, 3, 60, 80), generator=torch.Generator().manual_seed(2)).cuda()
        for t in (1, 2, 3):
            opt.zero_grad()
            images = BlendPointCloud(_info(sc, ns, shared_texels_in_order=True))
            (net(images) - target).square().mean().backward()
            if not runs:
                _check_chain(ns, sc, net, target, texture, confidence)
            if t == 1:
                first.append([p.grad.clone() for p in params[:2]])
            before = [p.detach().double().cpu().numpy().reshape(-1) for p in params]
            moments = [[x.double().cpu().numpy().reshape(-1) for x in opt.moments(p)] if p in opt.state else None for p in params]
            opt.step()
            if runs:
                continue
            gs = [p.grad.double().cpu().numpy().reshape(-1) for p in params]
            norm = np.sqrt(sum((g ** 2).sum() for g in gs))
            factor = min(1.0, np.float64(np.float32(0.05)) / (norm + 1e-6))
            got = opt.grad_norm.cpu().numpy()
            assert abs(got[0] - norm) <= 2.0 ** -23 * norm and abs(got[1] - factor) <= 2.0 ** -23 * factor
            for i, p in enumerate(params):
                group = opt.param_groups[0 if i < 2 else 1]
                m, v = moments[i] or (np.zeros(p.numel()), np.zeros(p.numel()))
                w, _, _, terms = ref.step(before[i], gs[i], m, v, t, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                                          float(got[1]))
                err = np.abs(p.detach().double().cpu().numpy().reshape(-1) - w)
                assert (err <= 2.0 ** -24 * (4 * np.abs(before[i]) + 24 * terms)).all()
        runs.append(None)
    assert all(torch.equal(a, b) for a, b in zip(*first))


def _check_chain(ns, sc, net, target, texture, confidence):
    """Gradients of the shared texels against those of the same chain with torch's indexing in the lookup's place: sums of the same
    float32 numbers (the splat gives the same per point), in another order."""
    from trips_amd.renderer import BlendPointCloud, NeuralScene
    n = sc.index.shape[0]
    index = ns.point_cloud_cuda.t_index.reshape(-1).long()
    own = [x.detach()[:, index].contiguous().requires_grad_() for x in (texture, confidence)]
    other = NeuralScene(texture=own[0], background_color=ns.texture.background_color, confidence=own[1],
                        position=ns.point_cloud_cuda.t_position, point_size=ns.point_cloud_cuda.t_point_size,
                        index=torch.arange(n, dtype=torch.int32, device="cuda").reshape(-1, 1), poses_se3=ns.poses.poses_se3,
                        intrinsics=ns.intrinsics.intrinsics)
    (net(BlendPointCloud(_info(sc, other))) - target).square().mean().backward(inputs=own)
    count = torch.bincount(index, minlength=TEXELS).double()
    for shared, per_point in zip((texture, confidence), own):
        g = per_point.grad.double()
        want = torch.zeros(shared.shape, dtype=torch.float64, device="cuda").index_add_(1, index, g)
        size = torch.zeros(shared.shape, dtype=torch.float64, device="cuda").index_add_(1, index, g.abs())
        assert ((shared.grad.double() - want).abs() <= (count + 2) * 2.0 ** -24 * size).all()
