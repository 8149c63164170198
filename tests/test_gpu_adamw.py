"""AdamW and the gradients' norm through the public classes, against the formulas in double precision.

Bounds are counted in roundings of float32 (2^-24 each). m: the products with beta1 and 1 - beta1 (each constant rounded as
well) and their sum, 4 of |beta1 m| + |(1 - beta1) g|, and 2 more with a factor on g. v: 6 of itself, 4 more with a factor on
g, whose rounding counts twice. The update: those of m on its terms, half of v's under the root, and 10 for the root, the
constants, the product with the root's correction, the sum with eps, the quotient and the product with the rate; the weight: its
own two and the last sum. 16-bit types add half a step of their own, eps / 2 of the value (and the least step's half)."""
import numpy as np
import pytest
import torch

from tests import optim_reference as ref
from trips_amd import abi

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = (1, 3, 255, 256, 257, 1023, 4097, 70001)


def _numbers(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def _half_step(dtype, value):
    if dtype is torch.float32:
        return 0.0
    info = torch.finfo(dtype)
    return np.abs(value) * info.eps / 2 * (1 + 4 * U) + info.smallest_normal * info.eps / 2


def _tensors(sizes, weights, grads, seed, offset=0):
    """Parameters and gradients; with an offset each begins that many elements behind an aligned address."""
    g = torch.Generator().manual_seed(seed)
    params, gs = [], []
    for n in sizes:
        w = torch.randn(n, generator=g) * 0.1
        x = torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g) * 3) * 0.01
        wide, wide_g = torch.zeros(n + offset, dtype=TYPES[weights], device="cuda"), torch.zeros(n + offset, dtype=TYPES[grads], device="cuda")
        wide[offset:], wide_g[offset:] = w.to(TYPES[weights]), x.to(TYPES[grads])
        params.append(torch.nn.Parameter(wide[offset:]))
        gs.append(wide_g[offset:])
    return params, gs


def _check_step(opt, before, params, gs, t, factor=1.0, places=None, seed=0):
    """One step's results against the formulas, from what was there before it. `factor` is the float32 one."""
    extra = 0 if factor == 1.0 else 2
    for i, (p, g) in enumerate(zip(params, gs)):
        group = next(q for q in opt.param_groups if any(p is x for x in q["params"]))
        w0, m0, v0 = before[i]
        w, m, v, terms = ref.step(w0, _numbers(g), m0, v0, t, group["lr"], group["betas"], group["eps"], group["weight_decay"], factor)
        b1 = group["betas"][0]
        parts = b1 * np.abs(m0) + (1 - b1) * np.abs(_numbers(g) * factor)
        st = opt.state[p]
        assert int(st["step"]) == t
        if "first_scale" not in st:
            got_m, got_v = _numbers(st["first_moment"]), _numbers(st["second_moment"])
            assert (np.abs(got_m - m) <= (4 + extra) * U * parts + 1e-45).all()
            assert (np.abs(got_v - v) <= (6 + 2 * extra) * U * v + 1e-44).all()
        else:
            bits = ref.mix(np.uint64(places[i]) + np.arange(p.numel(), dtype=np.uint64) ^ ref.mix(seed + t * 0x9E3779B9))
            for name, x, r, kind in (("first", m, bits & np.uint64(0xFFFF), (3, 7, 448.0, False)),
                                     ("second", v, bits >> np.uint64(16), (2, 15, 57344.0, True))):
                codes, scales, margin = ref.encode(x, r.astype(np.float64), *kind)
                assert margin > 2.0 ** -30  # (no element so near a border that double rounding counts)
                got = st[name + "_moment"].view(torch.uint8).reshape(-1).cpu().numpy()
                np.testing.assert_array_equal(st[name + "_scale"].cpu().numpy(), scales)
                np.testing.assert_array_equal(got, codes, err_msg=name)
        bound = U * (3 * np.abs(w0) + (4 + extra + 3 + extra + 10) * terms + np.abs(w)) + _half_step(p.dtype, w)
        err = np.abs(_numbers(p) - w)
        assert (err <= bound).all(), (i, (err / bound).max())


def _state(opt, params):
    out = []
    for p in params:
        st = opt.state.get(p)
        if not st:
            out.append((_numbers(p), np.zeros(p.numel()), np.zeros(p.numel())))
        elif "first_scale" in st:
            m = ref.decode(st["first_moment"].view(torch.uint8).reshape(-1).cpu().numpy(), st["first_scale"].cpu().numpy(), 3, 7)
            v = ref.decode(st["second_moment"].view(torch.uint8).reshape(-1).cpu().numpy(), st["second_scale"].cpu().numpy(), 2, 15)
            out.append((_numbers(p), m, v))
        else:
            out.append((_numbers(p), _numbers(st["first_moment"]), _numbers(st["second_moment"])))
    return out


def _places(params):
    at, out = 0, []
    for p in params:
        out.append(at)
        at += -(-p.numel() // 256) * 256
    return out


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("weights,grads", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"),
                                           ("f16", "f16"), ("f16", "f32"), ("bf16", "f16"), ("f16", "bf16")])
def test_three_steps(bits, weights, grads):
    from trips_amd.adamw import AdamW
    params, gs = _tensors(SIZES, weights, grads, 1)
    opt = AdamW(params, lr=3e-3, weight_decay=0.02, state_bits=bits, min_8bit_size=0, seed=77)
    for t in (1, 2, 3):
        before = _state(opt, params)
        opt.step(grads=dict(zip(params, gs)))
        _check_step(opt, before, params, gs, t, places=_places(params), seed=77)
        for g in gs:
            g.mul_(-0.5)  # (exact)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 3])
def test_odd_addresses_and_what_lies_beside(bits, offset):
    """Tensors that begin at any element; what lies before and behind them in the buffer stays."""
    from trips_amd.adamw import AdamW
    sizes = (1, 5, 255, 1026, 5001)
    total = sum(sizes) + offset + 7
    rng = torch.Generator().manual_seed(3)
    for weights, grads in ((torch.float32, torch.float32), (torch.bfloat16, torch.float16)):
        flat, flat_g = torch.randn(total, generator=rng).to(weights).cuda(), torch.randn(total, generator=rng).to(grads).cuda()
        guard = flat.clone()
        params, gs, at = [], [], offset
        for n in sizes:
            params.append(torch.nn.Parameter(flat[at:at + n]))
            gs.append(flat_g[at:at + n])
            at += n
        opt = AdamW(params, state_bits=bits, min_8bit_size=0)
        before = _state(opt, params)
        opt.step(grads=dict(zip(params, gs)))
        _check_step(opt, before, params, gs, 1, places=_places(params))
        assert torch.equal(flat[:offset], guard[:offset]) and torch.equal(flat[at:], guard[at:])


def test_many_tensors_groups_and_mixed_states():
    """More tensors than a launch holds, more sets of options than it holds, 8-bit and 32-bit states side by side."""
    from trips_amd.adamw import AdamW
    sizes = [1 + (i * 37) % 900 for i in range(97)]
    params, gs = _tensors(sizes, "f32", "f32", 5)
    groups = [dict(params=params[i::12], lr=1e-3 * (i + 1), betas=(0.9 - 0.05 * i, 0.99), eps=1e-6, weight_decay=0.01 * i)
              for i in range(12)]
    opt = AdamW(groups, state_bits=8, min_8bit_size=400, seed=9)
    in_call = [p for g in groups for p in g["params"]]
    gs_of = {p: g for p, g in zip(params, gs)}
    places = dict(zip(in_call, _places(in_call)))
    for t in (1, 2):
        before = _state(opt, params)
        opt.step(grads=gs_of)
        _check_step(opt, before, params, gs, t, places=[places[p] for p in params], seed=9)
    assert sum("first_scale" in opt.state[p] for p in params) == sum(n >= 400 for n in sizes)


def test_parameters_own_gradients_absent_and_empty_ones():
    from trips_amd.adamw import AdamW
    params, gs = _tensors((10, 0, 300), "f32", "f32", 6)
    params[0].grad, params[1].grad = gs[0], gs[1]
    opt = AdamW(params)
    before = _state(opt, params)
    opt.step()
    _check_step(opt, before[:1], params[:1], gs[:1], 1)
    assert params[2] not in opt.state and np.array_equal(_numbers(params[2]), before[2][0])
    assert int(opt.state[params[1]]["step"]) == 1
    opt.zero_grad()
    opt.step()  # nothing to do
    assert int(opt.state[params[0]]["step"]) == 1


@pytest.mark.parametrize("copy", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_copy_is_the_weight_before_its_rounding(copy, bits):
    from trips_amd.adamw import AdamW
    params, gs = _tensors((257, 1030), "f32", "bf16", 7)
    copies = [torch.full((p.numel() + 2,), 7.0, dtype=TYPES[copy], device="cuda") for p in params]
    opt = AdamW(params, state_bits=bits, min_8bit_size=0)
    for p, c in zip(params, copies):
        opt.set_copy(p, c[1:-1])
    opt.step(grads=dict(zip(params, gs)))
    for p, c in zip(params, copies):
        assert torch.equal(c[1:-1], p.detach().to(TYPES[copy]))
        assert float(c[0]) == 7.0 and float(c[-1]) == 7.0


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_and_loss_scale(bits):
    from trips_amd.adamw import AdamW, grad_norm
    params, gs = _tensors(SIZES, "f32", "bf16", 8)
    for g in gs:
        g.mul_(512.0)
    opt = AdamW(params, state_bits=bits, min_8bit_size=0, max_grad_norm=0.25, loss_scale=512.0, seed=4)
    norm = np.sqrt(sum((_numbers(g) ** 2).sum() for g in gs)) / 512
    want = np.array([norm, min(1.0, 0.25 / (norm + 1e-6)) / 512])
    assert want[1] * 512 < 1
    before = _state(opt, params)
    opt.step(grads=dict(zip(params, gs)))
    got = opt.grad_norm.cpu().numpy()
    assert (np.abs(got - want) <= 1.01 * U * np.abs(want)).all()
    _check_step(opt, before, params, gs, 1, factor=float(got[1]), places=_places(params), seed=4)
    assert torch.equal(grad_norm(gs, 0.25, 512.0), opt.grad_norm)
    # the same norm handed over
    before = _state(opt, params)
    given = grad_norm(gs, 0.5, 512.0)
    opt.step(grads=dict(zip(params, gs)), grad_norm=given)
    _check_step(opt, before, params, gs, 2, factor=float(given[1]), places=_places(params), seed=4)
    # a loss scale alone
    opt.max_grad_norm = 0.0
    before = _state(opt, params)
    opt.step(grads=dict(zip(params, gs)))
    assert opt.grad_norm is None
    _check_step(opt, before, params, gs, 3, factor=1.0 / 512, places=_places(params), seed=4)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_with_nonfinite_gradients_are_skipped(bad, bits):
    from trips_amd.adamw import AdamW
    params, gs = _tensors((300, 5000), "f32", "f16", 9)
    copy = params[1].detach().clone()
    opt = AdamW(params, state_bits=bits, min_8bit_size=0, skip_nonfinite=True)
    opt.set_copy(params[1], copy)
    given = dict(zip(params, gs))
    opt.step(grads=given)
    kept = [{k: v.clone() for k, v in opt.state[p].items()} for p in params]
    weights = [p.detach().clone() for p in params]
    gs[1][4999] = bad
    for _ in range(2):
        opt.step(grads=given)
        assert not np.isfinite(opt.grad_norm.cpu().numpy()[1])
        for p, st, w in zip(params, kept, weights):
            assert torch.equal(p, w) and all(torch.equal(opt.state[p][k].view(torch.uint8) if v.element_size() == 1 else opt.state[p][k],
                                                         v.view(torch.uint8) if v.element_size() == 1 else v) for k, v in st.items())
    assert torch.equal(copy, params[1])
    gs[1][4999] = 1.0
    before = _state(opt, params)
    opt.step(grads=given)
    _check_step(opt, before, params, gs, 2, places=_places(params))


def test_nonfinite_moments_of_8_bits_stay_with_their_element():
    from trips_amd.adamw import AdamW
    params, gs = _tensors((600,), "f32", "f32", 10)
    gs[0][5], gs[0][300] = float("inf"), float("nan")
    opt = AdamW(params, state_bits=8, min_8bit_size=0)
    before = _state(opt, params)
    opt.step(grads={params[0]: gs[0]})
    m, v = (x.cpu().numpy() for x in opt.moments(params[0]))
    bad = np.zeros(600, dtype=bool)
    bad[[5, 300]] = True
    assert np.isnan(m[bad]).all() and np.isnan(v[bad]).all() and np.isfinite(m[~bad]).all() and np.isfinite(v[~bad]).all()
    gs[0][bad] = 0.0
    clean, _ = _tensors((600,), "f32", "f32", 10)
    other = AdamW(clean, state_bits=8, min_8bit_size=0)
    other.step(grads={clean[0]: gs[0]})
    assert torch.equal(clean[0][torch.as_tensor(~bad)], params[0][torch.as_tensor(~bad)])
    m2, v2 = (x.cpu().numpy() for x in other.moments(clean[0]))
    np.testing.assert_array_equal(m[~bad], m2[~bad])
    np.testing.assert_array_equal(v[~bad], v2[~bad])
    assert before


@pytest.mark.parametrize("value", [0.0, 1e-30, 3e-20, 1e4, 1e11])
def test_8_bits_over_the_range_of_gradients(value):
    """Blocks of zeros, of tiny and of huge numbers, and one element far above the others: no positive v becomes zero."""
    from trips_amd.adamw import AdamW
    params, gs = _tensors((512,), "f32", "f32", 11)
    gs[0].mul_(value)
    if value:
        gs[0][7] = value * 1e7
    opt = AdamW(params, state_bits=8, min_8bit_size=0, eps=1e-8)
    for t in (1, 2):
        before = _state(opt, params)
        opt.step(grads={params[0]: gs[0]})
        _check_step(opt, before, params, gs, t, places=[0])
        v = opt.moments(params[0])[1].cpu().numpy()
        square = _numbers(gs[0]) ** 2
        if 1e-40 < value ** 2 < 1e40:
            assert (v[square > 0] > 0).all()
        assert np.isfinite(_numbers(params[0])).all()


def test_rounding_to_8_bits_keeps_small_changes_on_average():
    """v of a constant gradient over 400 steps of 1 / 1000: its mean follows the exact average. Each element's v is that average
    times a mean-one noise; with steps of at most a quarter of a value, and increments of less than one step that are each rounded
    up with the probability that keeps the mean, the noise's relative deviation after 400 steps is below one, so that the mean of
    2^16 elements is within 6 / 2^8 of it."""
    from trips_amd.adamw import AdamW
    n = 1 << 16
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = torch.full((n,), 0.5, device="cuda")
    opt = AdamW([p], lr=0.0, state_bits=8, min_8bit_size=0)
    for _ in range(400):
        opt.step()
    m, v = opt.moments(p)
    assert abs(float(v.double().mean()) / (0.25 * (1 - 0.999 ** 400)) - 1) < 6 / 256
    assert abs(float(m.double().mean()) / 0.5 - 1) < 6 / 256


def test_repeatable_and_seeded():
    from trips_amd.adamw import AdamW
    out = []
    for seed in (1, 1, 2):
        params, gs = _tensors((5000,), "f32", "f32", 12)
        opt = AdamW(params, state_bits=8, min_8bit_size=0, seed=seed, max_grad_norm=1.0)
        for _ in range(3):
            opt.step(grads={params[0]: gs[0]})
        out.append((params[0].detach().clone(), opt.moments(params[0])[1]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    assert not torch.equal(out[0][1], out[2][1])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("weights", ["f32", "bf16"])
def test_state_dict_goes_on_bit_for_bit(bits, weights):
    from trips_amd.adamw import AdamW
    params, gs = _tensors((300, 5000), weights, "f32", 13)
    opt = AdamW(params, state_bits=bits, min_8bit_size=1000, max_grad_norm=1.0, seed=3)
    given = dict(zip(params, gs))
    for _ in range(2):
        opt.step(grads=given)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW(twins, max_grad_norm=1.0, seed=3)
    other.load_state_dict(opt.state_dict())
    for p, q in zip(params, twins):
        assert all(opt.state[p][k].dtype == v.dtype and v.device == q.device for k, v in other.state[q].items())
        assert other.state[q]["first_moment"].data_ptr() != opt.state[p]["first_moment"].data_ptr()
    opt.step(grads=given)
    other.step(grads=dict(zip(twins, gs)))
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(p), other.moments(q)))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays_with_its_counts(bits):
    """A step recorded into a graph and replayed, with eager work and other steps in between, against eager steps."""
    from trips_amd.adamw import AdamW
    both = []
    for _ in range(2):
        params, gs = _tensors((300, 9000, 17), "f32", "f32", 14)
        both.append((params, gs, AdamW(params, state_bits=bits, min_8bit_size=0, max_grad_norm=0.5, seed=5)))
    (params, gs, opt), (twins, gs2, eager) = both
    opt.step(grads=dict(zip(params, gs)))
    eager.step(grads=dict(zip(twins, gs2)))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    given = dict(zip(params, gs))
    with torch.cuda.graph(graph, stream=side):
        opt.step(grads=given)
    for k in range(4):
        for a, b in zip(gs, gs2):
            a.mul_(0.5), b.mul_(0.5)
        if k == 3:  # one that is skipped
            gs[1][0] = gs2[1][0] = float("inf")
        graph.replay()
        eager.step(grads=dict(zip(twins, gs2)))
        torch.cuda.synchronize()
        for p, q in zip(params, twins):
            assert torch.equal(p, q), k
            assert int(opt.state[p]["step"]) == int(eager.state[q]["step"]) == min(k + 2, 4)
            assert all(torch.equal(a, b) for a, b in zip(opt.moments(p), eager.moments(q)))
        junk = torch.randn(100_000, device="cuda").sort()[0]
        torch.cuda.synchronize()
        del junk


def test_first_steps_cannot_be_captured_and_captured_ones_outlive_larger_steps():
    """A captured step of one parameter of two; an eager step of both in between, and much else allocated."""
    from trips_amd.adamw import AdamW
    params, gs = _tensors((3000, 5000), "f32", "f32", 17)
    opt = AdamW(params, max_grad_norm=0.5)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        with pytest.raises(RuntimeError, match="captured"):
            opt.step(grads={params[0]: gs[0]})
        graph.capture_end()
    torch.cuda.synchronize()
    opt.step(grads={params[0]: gs[0]})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step(grads={params[0]: gs[0]})
    opt.step(grads=dict(zip(params, gs)))
    opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4, device="cuda")) for _ in range(100)]))
    for p in opt.param_groups[1]["params"]:
        p.grad = torch.ones_like(p)
    opt.step()
    junk = [torch.full((64, 1024), float("nan"), device="cuda") for _ in range(50)]
    for t in (3, 4):
        before = _state(opt, params[:1])
        graph.replay()
        torch.cuda.synchronize()
        norm = np.sqrt((_numbers(gs[0]) ** 2).sum())
        _check_step(opt, before, params[:1], gs[:1], t, factor=float(np.float32(min(1.0, 0.5 / (norm + 1e-6)))))
    assert all(torch.isnan(j).all() for j in junk)


def test_copies_of_the_optimiser():
    import copy
    from trips_amd.adamw import AdamW
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.full_like(p, 0.5)
    opt = AdamW([p], max_grad_norm=0.25, state_bits=8, min_8bit_size=0, seed=6)
    opt.step()
    twin = copy.deepcopy(opt)
    q = twin.param_groups[0]["params"][0]
    assert q is not p and torch.equal(p, q) and (twin.max_grad_norm, twin.seed) == (0.25, 6)
    q.grad = p.grad.clone()
    opt.step(), twin.step()
    assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(opt.moments(p), twin.moments(q)))


def test_a_tensor_of_more_than_2_31_elements():
    """The last elements of 2^31 + 1000, the others zeros: offsets pass 32 bits, places of the rounding wrap at 2^32 no sooner."""
    from trips_amd.adamw import AdamW
    n, tail = (1 << 31) + 1000, 1300
    w, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    rng = torch.Generator().manual_seed(18)
    w[-tail:], g[-tail:] = (torch.randn(tail, generator=rng).to(torch.bfloat16).cuda() for _ in range(2))
    p = torch.nn.Parameter(w)
    opt = AdamW([p], state_bits=8, max_grad_norm=1.0, seed=3)
    before = w[-tail:].double().cpu().numpy()
    opt.step(grads={p: g})
    gd = g[-tail:].double().cpu().numpy()
    norm = np.sqrt((gd ** 2).sum())
    got = opt.grad_norm.cpu().numpy()
    assert abs(got[0] - norm) <= 1.01 * U * norm
    want, m, v, terms = ref.step(before, gd, np.zeros(tail), np.zeros(tail), 1, 1e-3, (0.9, 0.999), 1e-8, 1e-2, float(got[1]))
    bound = U * (3 * np.abs(before) + 21 * terms + np.abs(want)) + _half_step(torch.bfloat16, want)
    assert (np.abs(w[-tail:].double().cpu().numpy() - want) <= bound).all()
    # the moments of the last whole block and of the rest, rounded by their places
    first = n - n % 256 - 256
    skip = tail - (n - first)
    bits = ref.mix(np.arange(first, n, dtype=np.uint64) ^ ref.mix(3 + 0x9E3779B9))
    for name, x, r, kind in (("first", m, bits & np.uint64(0xFFFF), (3, 7, 448.0, False)), ("second", v, bits >> np.uint64(16), (2, 15, 57344.0, True))):
        codes, scales, margin = ref.encode(x[skip:], r.astype(np.float64), *kind)
        assert margin > 2.0 ** -30
        st = opt.state[p]
        np.testing.assert_array_equal(st[name + "_scale"][-2:].cpu().numpy(), scales)
        np.testing.assert_array_equal(st[name + "_moment"].view(torch.uint8)[first:].cpu().numpy(), codes)
    assert not w[:100_000].any() and not w[1 << 30:(1 << 30) + 100_000].any()


def test_another_stream():
    from trips_amd.adamw import AdamW
    params, gs = _tensors((5000, 200_000), "f32", "f32", 15)
    opt = AdamW(params, max_grad_norm=1.0)
    before = _state(opt, params)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for g in gs:
            g.mul_(4.0)
        opt.step(grads=dict(zip(params, gs)))
        factor = float(opt.grad_norm[1])
    side.synchronize()
    _check_step(opt, before, params, gs, 1, factor=factor)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes", [(0,), (1,), (4095, 4096, 4097), tuple(range(1, 260)), (2_000_003, 17)])
def test_norm(dtype, sizes):
    """More tensors than a launch holds; the sum is in double, so the result is that of double rounded once (a count of at most
    2^22 terms leaves 2^-31 of it to the order)."""
    from trips_amd.adamw import grad_norm
    g = torch.Generator().manual_seed(16)
    flat = (torch.randn(sum(sizes) + 1, generator=g) * 3).to(TYPES[dtype]).cuda()
    views, at = [], 1
    for n in sizes:
        views.append(flat[at:at + n])
        at += n
    norm = np.sqrt(sum((_numbers(x) ** 2).sum() for x in views))
    for max_norm, scale in ((0.0, 1.0), (1.5, 1.0), (1e9, 8.0)):
        got = grad_norm(views, max_norm, scale).cpu().numpy().astype(np.float64)
        factor = (min(1.0, max_norm / (norm / scale + 1e-6)) if max_norm else 1.0) / scale
        want = np.array([norm / scale, factor])
        assert (np.abs(got - want) <= 1.01 * U * want).all()


def test_norm_of_large_and_small_numbers_and_of_nonfinite_ones():
    from trips_amd.adamw import grad_norm
    x = torch.full((1000,), 1e30, device="cuda")
    assert abs(float(grad_norm([x])[0]) / (1e30 * np.sqrt(1000)) - 1) < 1e-6  # squares pass float's range
    x = torch.full((1000,), 1e-30, device="cuda")
    assert abs(float(grad_norm([x])[0]) / (1e-30 * np.sqrt(1000)) - 1) < 1e-6
    for bad in (float("inf"), float("nan"), -float("inf")):
        x = torch.ones(70_000, device="cuda")
        x[69_999] = bad
        got = grad_norm([torch.ones(5, device="cuda"), x], 1.0).cpu().numpy()
        assert not np.isfinite(got[0]) and np.isnan(got[1])
    assert grad_norm([torch.zeros(10, device="cuda")], 1.0).tolist() == [0.0, 1.0]


def test_hooks_closures_versions_and_schedulers():
    from trips_amd.adamw import AdamW
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = AdamW([p], lr=0.1)
    seen = []
    before, after = opt.register_step_pre_hook(lambda *a: seen.append("before")), opt.register_step_post_hook(lambda *a: seen.append("after"))

    def closure():
        seen.append("loss")
        opt.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss
    assert float(opt.step(closure)) == 8.0 and seen == ["before", "loss", "after"]
    before.remove(), after.remove()
    with torch.profiler.profile() as profile:
        opt.step(closure)
    assert seen == ["before", "loss", "after", "loss"]
    assert any("AdamW" in e.name for e in profile.events())
    scheduler = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    opt.step(closure)
    scheduler.step()
    assert opt.param_groups[0]["lr"] == 0.05
    loss = (p * p).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals():
    from trips_amd._lib import TripsError
    from trips_amd.adamw import AdamW, grad_norm
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    for kw in (dict(lr=-1), dict(eps=-1), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(weight_decay=-1), dict(state_bits=16),
               dict(max_grad_norm=-1), dict(loss_scale=0.0), dict(lr=float("nan")), dict(loss_scale=float("inf"))):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    opt = AdamW([p])
    with pytest.raises(RuntimeError, match="elements"):
        opt.step(grads={p: torch.zeros(7, device="cuda")})
    with pytest.raises(RuntimeError, match="float64"):
        opt.step(grads={p: torch.zeros(8, device="cuda", dtype=torch.float64)})
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step(grads={p: torch.zeros(8, device="cuda").to_sparse()})
    with pytest.raises(RuntimeError, match="one device"):
        opt.step(grads={p: torch.zeros(8)})
    with pytest.raises(RuntimeError, match="contiguous"):
        AdamW([q := torch.nn.Parameter(torch.zeros(8, 8, device="cuda").t())]).step(grads={q: torch.zeros(8, 8, device="cuda")})
    with pytest.raises(RuntimeError, match="float32"):
        AdamW([q := torch.nn.Parameter(torch.zeros(8, device="cuda", dtype=torch.float64))]).step(grads={q: torch.zeros(8, device="cuda")})
    with pytest.raises(ValueError, match="two float32"):
        opt.step(grads={p: torch.zeros(8, device="cuda")}, grad_norm=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError, match="copy"):
        opt.set_copy(p, torch.zeros(9, device="cuda"))
    with pytest.raises(ValueError):
        grad_norm([])
    with pytest.raises(TripsError):
        grad_norm([torch.zeros(8, device="cuda")], loss_scale=0.0)
    opt.param_groups[0]["lr"] = float("nan")
    with pytest.raises(TripsError, match="lr"):
        opt.step(grads={p: torch.zeros(8, device="cuda")})
    assert float(p.detach().abs().sum()) == 0.0
    assert abi.TRIPS_MOMENT_BLOCK == ref.BLOCK
