"""A table's cross entropy and its gradients against numpy in double precision; the bounds are loss_reference.Loss's."""
import numpy as np
import pytest
import torch

from tests.loss_reference import U, Loss, within
from trips_amd.table_loss import table_cross_entropy

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _inputs(n, t, c, dtype, padding=0.0, index=torch.int64, seed=0, pad=0, spread=2.0):
    """Rows lean towards their targets; `pad` elements lie between two rows of either matrix."""
    rng = np.random.default_rng(seed + n + 7 * t + 31 * c)
    w = rng.normal(size=(t, c + pad)) * spread / np.sqrt(c)
    target = (rng.random(n) ** 2 * t).astype(np.int64)
    x = rng.normal(size=(n, c + pad)) + w[target]
    target[rng.random(n) < padding] = rng.choice([-1, t, -100, t + 5])
    x, w = (torch.as_tensor(a, dtype=TYPES[dtype], device="cuda")[:, :c] for a in (x, w))
    return x.requires_grad_(), w.requires_grad_(), torch.as_tensor(target, dtype=index, device="cuda")


def _weights(reduction, target, t, rng):
    inside = ((target >= 0) & (target < t)).cpu().numpy().reshape(-1)
    if reduction == "none":
        g = torch.as_tensor(rng.normal(size=inside.size), dtype=torch.float32, device="cuda")
        return g, g.double().cpu().numpy() * inside
    g = torch.tensor(1.5, device="cuda")
    return g, inside * (1.5 / (max(1, inside.sum()) if reduction == "mean" else 1))


def _check(x, w, target, scale=1.0, reduction="none", seed=3):
    rng = np.random.default_rng(seed)
    upstream, weights = _weights(reduction, target, w.shape[0], rng)
    want = Loss(x, w, target, scale, weights)
    loss = table_cross_entropy(x, w, target, scale=scale, reduction=reduction)
    assert loss.dtype == torch.float32
    with torch.no_grad():
        assert torch.equal(loss, table_cross_entropy(x, w, target, scale=scale, reduction=reduction))
    d_rows, d_table = torch.autograd.grad(loss, (x, w), upstream)
    if reduction == "none":
        within(loss, want.losses, want.loss_bound, "loss")
        assert (loss.detach().cpu().numpy()[~want.counts] == 0).all()
    else:
        by = max(1, want.counts.sum()) if reduction == "mean" else 1
        total = want.losses.sum() / by
        within(loss, np.array(total), np.array(want.loss_bound.sum() / by + 2.0 ** -24 * abs(total)), "loss")
    assert d_rows.dtype == x.dtype and d_table.dtype == w.dtype
    within(d_rows, want.d_rows, want.d_rows_bound, "d_rows")
    within(d_table, want.d_table, want.d_table_bound, "d_table")
    assert (d_rows.cpu().numpy()[~want.counts] == 0).all() if x.dtype != torch.bfloat16 else (d_rows[torch.as_tensor(~want.counts)] == 0).all()
    return loss, d_rows, d_table


SIZES = [(1, 1, 1), (1, 5, 3), (3, 2, 8), (1, 3000, 1024), (2, 257, 64), (16, 700, 72), (25, 5000, 64), (31, 129, 33), (33, 4099, 256), (130, 300, 40), (257, 128, 16),
         (255, 256, 64), (300, 1000, 100), (513, 777, 65), (700, 20, 4), (1000, 150, 16), (64, 511, 2050), (128, 20_000, 32), (1023, 1500, 200)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,t,c", SIZES)
def test_sizes(n, t, c, dtype):
    _check(*_inputs(n, t, c, dtype))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("padding", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_padding_and_reductions(dtype, reduction, padding, index):
    _check(*_inputs(150, 333, 48, dtype, padding, index), reduction=reduction)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", [0.0, 0.05, 3.0, -1.0, -0.3])
def test_scales(dtype, scale):
    _check(*_inputs(70, 290, 56, dtype, 0.1), scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [16_384, 16_400, 9_000, 20_480, 20_481, 21_530])
def test_many_rows(n, dtype):
    _check(*_inputs(n, 60, 24, dtype, 0.4), reduction="mean")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,t,c,pad", [(3, 17_000, 500, 0), (32, 9000, 70, 1), (33, 9001, 70, 0), (64, 9000, 140, 0), (65, 8500, 130, 5), (600, 33, 1000, 0), (40, 97, 2000, 1), (500, 31, 700, 0),
                                       (2, 65, 9, 0)])
def test_few_rows_or_few_tiles(n, t, c, pad, dtype):
    _check(*_inputs(n, t, c, dtype, 0.2 if n > 3 else 0, pad=pad), scale=0.7, reduction="sum")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,t,c", [(1, 70_001, 8), (3, 300_000, 4), (30, 66_000, 5), (64, 140_000, 4), (65, 140_000, 4)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_few_rows_of_very_many_entries(n, t, c, dtype, reduction):
    _check(*_inputs(n, t, c, dtype, 0.3 if n > 3 else 0), reduction=reduction)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,t,c,pad", [(20_000, 150, 16, 0), (16_384, 2, 100, 3), (12_001, 65, 33, 0), (3000, 7, 700, 1), (9000, 129, 257, 0)])
def test_few_entries_of_many_rows(n, t, c, pad, dtype):
    """The table's gradient is a sum over many rows: cut into parts."""
    _check(*_inputs(n, t, c, dtype, 0.3, pad=pad), scale=-0.7, reduction="none" if t == 65 else "mean")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_more_than_a_million_rows(dtype):
    _check(*_inputs(1_100_000, 40, 6, dtype, 0.3), reduction="mean")


def test_no_rows_and_no_entries():
    for dtype in TYPES.values():
        x, w = torch.zeros(0, 8, dtype=dtype, device="cuda", requires_grad=True), torch.randn(5, 8, device="cuda").to(dtype).requires_grad_()
        none = torch.zeros(0, dtype=torch.int64, device="cuda")
        for reduction in ("none", "sum", "mean"):
            loss = table_cross_entropy(x, w, none, reduction=reduction)
            assert loss.shape == ((0,) if reduction == "none" else ()) and float(loss.detach().sum()) == 0
            d_rows, d_table = torch.autograd.grad(loss.sum(), (x, w))
            assert d_rows.shape == x.shape and (d_table == 0).all()
        rows = torch.randn(3, 8, device="cuda").to(dtype).requires_grad_()
        nothing = torch.zeros(0, 8, dtype=dtype, device="cuda", requires_grad=True)
        loss = table_cross_entropy(rows, nothing, torch.zeros(3, dtype=torch.int32, device="cuda"))
        d_rows, d_table = torch.autograd.grad(loss, (rows, nothing))
        assert float(loss.detach()) == 0 and (d_rows == 0).all() and d_table.shape == (0, 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad", [1, 8, 13])
@pytest.mark.parametrize("c", [64, 57])
def test_strided_rows(dtype, pad, c):
    _check(*_inputs(90, 400, c, dtype, 0.1, pad=pad))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_unaligned_and_transposed(dtype, shift):
    x, w, target = _inputs(65, 300, 64, dtype)
    flat = [torch.empty(m.numel() + shift, dtype=m.dtype, device="cuda") for m in (x, w)]
    moved = [f[shift:].view(m.shape).copy_(m.detach()).requires_grad_() for f, m in zip(flat, (x, w))]
    got = _check(*moved, target)
    for a, b in zip(got, _check(x, w, target)):
        assert torch.equal(a, b)
    turned = [m.detach().t().contiguous().t().requires_grad_() for m in (x, w)]
    for a, b in zip(got, _check(*turned, target)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,t,c,pad", [(40, 300, 57, 1), (40, 300, 62, 2), (300, 900, 33, 7), (9, 70, 3, 5), (600, 4000, 66, 2), (50, 200, 129, 3)])
def test_what_lies_behind_a_row(dtype, n, t, c, pad):
    """Elements between the rows hold anything; the same gradients as without them."""
    x, w, target = _inputs(n, t, c, dtype, 0.2)
    want = _check(x, w, target)
    wide = [torch.full((m.shape[0], c + pad), float("nan"), dtype=m.dtype, device="cuda") for m in (x, w)]
    views = [m[:, :c].copy_(a.detach()) for m, a in zip(wide, (x, w))]
    for m in views:
        assert m.stride(0) == c + pad
    for a, b in zip(_check_only(*views, target), want):
        assert torch.equal(a, b)


def test_rows_that_repeat():
    """One row of memory for all rows: read, its gradients summed by torch."""
    x, w, target = _inputs(1, 100, 16, "f32")
    target = torch.arange(40, device="cuda")
    loss = table_cross_entropy(x.expand(40, 16), w, target, reduction="sum")
    same = table_cross_entropy(x.detach().repeat(40, 1), w, target, reduction="sum")
    assert torch.equal(loss, same) and torch.autograd.grad(loss, x)[0].shape == x.shape


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_padding_holds_anything(dtype, bad):
    x, w, target = _inputs(140, 300, 40, dtype, 0.3)
    outside = (target < 0) | (target >= 300)
    clean = _check(x, w, target)
    x = x.detach().clone()
    x[outside] = bad
    for a, b in zip(_check_only(x, w, target), clean):
        assert torch.equal(a, b)


def _check_only(x, w, target, reduction="none"):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = table_cross_entropy(x, w, target, reduction=reduction)
    upstream, _ = _weights(reduction, target, w.shape[0], np.random.default_rng(3))
    return (loss, *torch.autograd.grad(loss, (x, w), upstream))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_row_without_numbers_leaves_the_others_theirs(dtype):
    """NaN in a row that counts: its loss and gradient are NaN, those of the other rows are not touched."""
    x, w, target = _inputs(140, 300, 40, dtype)
    loss, d_rows, _ = _check_only(x, w, target)
    y = x.detach().clone()
    y[17, 3] = float("nan")
    loss2, d_rows2, _ = _check_only(y, w, target)
    others = torch.arange(140, device="cuda") != 17
    assert torch.equal(loss[others], loss2[others]) and loss2[17].isnan()
    assert torch.equal(d_rows[others], d_rows2[others]) and d_rows2[17].isnan().any()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_gradient_without_a_number_is_its_own_rows(dtype):
    x, w, target = _inputs(140, 300, 40, dtype)
    loss = table_cross_entropy(x, w, target, reduction="none")
    g = torch.ones(140, device="cuda")
    want, = torch.autograd.grad(loss, (x,), g, retain_graph=True)
    for bad in (float("nan"), float("inf")):
        g[17] = bad
        got, = torch.autograd.grad(loss, (x,), g, retain_graph=True)
        others = torch.arange(140, device="cuda") != 17
        assert torch.equal(want[others], got[others]) and not torch.isfinite(got[17]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("all_masked", [False, True])
def test_entries_masked_with_the_lowest_value(dtype, all_masked):
    """A channel that is 1 in every row and holds the type's lowest value in masked entries: those have no part in the sum, and where
    there are no others, all have the same."""
    n, t, c = 50, 300, 16
    x, w, target = _inputs(n, t, c, dtype)
    x, w = x.detach().clone(), w.detach().clone()
    masked = torch.arange(t, device="cuda") % 3 > 0
    if all_masked:
        masked[:] = True
    target = torch.randint(0, t // 3, (n,), device="cuda") * 3
    x[:, -1], w[:, -1] = 1, 0
    w[masked, -1] = torch.finfo(w.dtype).min
    if all_masked:
        w[:, :-1] = 0
    x.requires_grad_(), w.requires_grad_()
    loss = table_cross_entropy(x, w, target, reduction="none")
    d_rows, d_table = torch.autograd.grad(loss.sum(), (x, w))
    logits = x.detach().double() @ w.detach().double().t()
    logp = torch.log_softmax(logits, 1)
    within(loss, -logp[torch.arange(n), target].cpu().numpy(), np.full(n, 1e-4), "loss")
    p = torch.softmax(logits, 1)
    p[torch.arange(n), target] -= 1
    u = max(torch.finfo(w.dtype).eps, 2.0 ** -16)
    within(d_table, (p.t() @ x.detach().double()).cpu().numpy(), (u * 4 * (p.abs().t() @ x.detach().double().abs())).cpu().numpy() + 1e-5, "d_table")
    if not all_masked:  # (the masked channel's own gradient is 0 times the lowest value)
        within(d_rows[:, :-1], (p @ w.detach().double())[:, :-1].cpu().numpy(), (u * 4 * (p.abs() @ w.detach().double().abs())[:, :-1]).cpu().numpy() + 1e-5, "d_rows")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_large_logits(dtype):
    _check(*_inputs(60, 200, 64, dtype, spread=60.0))


def _check_on_the_gpu(x, w, target, reduction="sum"):
    """For sizes that numpy would take long for: the oracle's products in double precision on the GPU. The bound is loss_reference.Loss's, with the
    largest error of any row's log probabilities: e of them, (terms + 8) 2 U for a sum of so many terms, half a step of the type where d_ij is held in it,
    half a step of the result."""
    (n, c), t = x.shape, w.shape[0]
    loss, d_rows, d_table = _check_only(x, w, target, reduction)
    inside = (target >= 0) & (target < t)
    i, u = inside.nonzero()[:, 0], torch.finfo(x.dtype).eps
    rows, table = x.detach()[i].double(), w.detach().double()
    p = rows @ table.t()
    size = float((rows.abs() @ table.t().abs()).max())
    at = torch.arange(i.numel(), device="cuda")
    p = torch.log_softmax(p, 1)
    total = -p[at, target[i]].sum()
    e = (4 * (c + 2) * size + 8 * size + 320 + t / 64 + 8) * U
    assert abs(float(loss.detach()) - float(total)) <= i.numel() * e + 4 * U * float(total)
    p.exp_()
    p[at, target[i]] -= 1
    p *= 1.5
    for got, a, b in ((d_rows[i], p, table), (d_table, p.t(), rows)):
        want, bound = a @ b, (u + 2 * e + (a.shape[1] + 16) * 2 * U) * (a.abs() @ b.abs()) + 1e-9
        off = (got.double() - want).abs() > bound
        assert not off.any() and not got.isnan().any(), f"{int(off.sum())} of {off.numel()} off"
    assert (d_rows[~inside] == 0).all()


LARGE = [(9000, 17_000, 8, 0), (300, 40_000, 40, 0), (600, 30_001, 66, 0), (200, 14_000, 1100, 0), (2000, 9000, 257, 0), (2049, 8193, 130, 3), (130, 66_000, 72, 0), (129, 70_000, 513, 1),
         (513, 33_000, 520, 8)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,t,c,pad", LARGE)
def test_large_tiles(n, t, c, pad, dtype):
    """Tiles of 256 x 256 in 16 bits, for the logits, the gradients or both, and the same sizes in 32."""
    _check_on_the_gpu(*_inputs(n, t, c, dtype, 0.2, pad=pad))


@pytest.mark.parametrize("n,t,c,dtype", [(70_000, 9000, 8, "bf16"), (66_000, 8300, 24, "f16"), (35_000, 8000, 12, "f32"), (150, 40_000, 1001, "bf16"), (140, 66_000, 513, "f16")])
def test_pieces_of_the_table(n, t, c, dtype):
    """More rows and entries than the logits' gradient of a piece holds, and (of odd channels) more entries than are copied at a time."""
    _check_on_the_gpu(*_inputs(n, t, c, dtype, 0.2))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gradients_against_differences(dtype):
    """The loss's own change along a direction: central differences of the kernel's losses, h = 2^-4 in a type with the steps for it,
    off by the third derivative's h^2 / 6 (logits' change d along the direction: at most 4 max|d|^3 h^2 / 6) and the losses' bound / h."""
    x, w, target = _inputs(20, 90, 32, "f32")
    x, w = (m.detach().to(TYPES[dtype]).requires_grad_() for m in (x, w))
    weights = np.ones(20)
    want = Loss(x, w, target, 1.0, weights)
    d_rows, d_table = torch.autograd.grad(table_cross_entropy(x, w, target, reduction="sum"), (x, w))
    g = torch.Generator(device="cuda").manual_seed(5)
    h = 2.0 ** -4
    for which, grad, bound in ((0, d_rows, want.d_rows_bound), (1, d_table, want.d_table_bound)):
        base = (x, w)[which].detach()
        direction = torch.randint(-1, 2, base.shape, device="cuda", generator=g).to(base.dtype)
        ends = [(base.double() + s * h * direction.double()).to(base.dtype) for s in (1, -1)]
        moved = (ends[0].double() - ends[1].double())  # (as far as the type let it move)
        losses = [float(table_cross_entropy(*((e, w) if which == 0 else (x, e)), target, reduction="none").double().sum()) for e in ends]
        along = float((grad.double() * moved).sum())
        change = (moved @ w.detach().double().t()) if which == 0 else (x.detach().double() @ moved.t())
        # (rounding makes the ends' middle another point than the base: the second derivative times that distance)
        middle = (ends[0].double() + ends[1].double()) / 2 - base.double()
        drift = (middle @ w.detach().double().t()) if which == 0 else (x.detach().double() @ middle.t())
        third = float((change.abs().amax(1) ** 3).sum()) * 4 / 24
        second = float((change.abs().amax(1) * drift.abs().amax(1)).sum()) * 2
        slack = float((torch.as_tensor(bound) * moved.abs().cpu()).sum()) + 2 * want.loss_bound.sum() * 2
        assert abs(losses[0] - losses[1] - along) <= third + second + slack, (losses, along, third, second, slack)


def test_same_bits_every_time_and_on_another_stream():
    x, w, target = _inputs(700, 3000, 96, "bf16", 0.2)
    want = _check_only(x, w, target, "mean")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            got = _check_only(x, w, target, "mean")
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,t,c", [(20_000, 150, 16), (40, 97, 2000), (30, 66_000, 5), (500, 31, 700), (300, 3000, 70), (600, 9000, 300)])
def test_same_bits_two_at_once(n, t, c, dtype):
    """Two calls on two streams at the same time, each with its own tensors, and again alone."""
    sets = [_inputs(n, t, c, dtype, 0.2, seed=s) for s in (1, 2)]
    alone = [(loss, *torch.autograd.grad(loss, (x, w))) for x, w, target in sets for loss in [table_cross_entropy(x, w, target)]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for stream, (x, w, target) in zip(streams, sets):
            with torch.cuda.stream(stream):
                loss = table_cross_entropy(x, w, target)
                got.append((loss, *torch.autograd.grad(loss, (x, w))))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for one, other in zip(got, alone) for a, b in zip(one, other))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,t,c", [(600, 33, 1000), (500, 31, 700), (4000, 20, 100), (40, 97, 2000), (65, 8500, 130), (20_000, 150, 16), (3, 17_000, 500), (300, 3000, 70), (700, 9001, 300),
                                   (7, 19, 2696)])
def test_workspaces_of_any_content(n, t, c, dtype):
    """What the allocator hands out for workspaces and results holds no numbers."""
    x, w, target = _inputs(n, t, c, dtype, 0.2)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    del [torch.full((1 << 27,), float("nan"), device="cuda")][:]
    for size in (1 << 8, 1 << 12, 1 << 16):  # (small blocks come from a pool of their own)
        del [torch.full((size,), float("nan"), device="cuda") for _ in range(64)][:]
    _check(x, w, target, reduction="mean")


def test_only_one_gradient():
    x, w, target = _inputs(100, 300, 32, "bf16", 0.2)
    _, d_rows, d_table = _check_only(x, w, target, "mean")
    up = torch.tensor(1.5, device="cuda")
    assert torch.equal(torch.autograd.grad(table_cross_entropy(x, w.detach(), target), x, up)[0], d_rows)
    assert torch.equal(torch.autograd.grad(table_cross_entropy(x.detach(), w, target), w, up)[0], d_table)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_steps(dtype):
    """Forward and backward in a graph, replayed with other inputs between eager calls on them."""
    x, w, target = _inputs(200, 900, 64, dtype, 0.2)
    x, w = x.detach(), w.detach()
    up = torch.tensor(1.5, device="cuda")

    def step(a, b):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        loss = table_cross_entropy(a, b, target)
        return (loss, *torch.autograd.grad(loss, (a, b), up))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(x, w)
    for i in range(4):
        x.copy_(torch.randn_like(x.float()))
        target[i * 3:i * 3 + 9] = -1 if i % 2 else i
        want = [o.detach().clone() for o in step(x, w)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_graphs_and_eager_calls():
    """Graphs of other sizes, replayed in turn: each has workspaces of its own."""
    sets, graphs = [_inputs(60, 500, 64, "bf16"), _inputs(90, 333, 40, "bf16", 0.5)], []
    for x, w, target in sets:
        table_cross_entropy(x, w, target)
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.no_grad(), torch.cuda.graph(graph, stream=side):
            graphs.append((graph, table_cross_entropy(x, w, target)))
    with torch.no_grad():
        want = [table_cross_entropy(*s) for s in sets]
    for _ in range(3):
        for (graph, got), x in zip(graphs, want):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got, x) for (_, got), x in zip(graphs, want))


def test_what_changed_before_the_gradients():
    """The rows that count and their targets are kept; the table is not, and refused where it was written to."""
    x, w, target = _inputs(20, 50, 16, "f32")
    want = torch.autograd.grad(table_cross_entropy(x, w, target), (x, w))
    loss = table_cross_entropy(x, w, target)
    with torch.no_grad():
        x.zero_(), target.zero_()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w), retain_graph=True), want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w), retain_graph=True), want))  # (and again)
    with torch.no_grad():
        w.add_(0)
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


def test_gradients_once():
    x, w, target = _inputs(20, 50, 16, "f32")
    d, = torch.autograd.grad(table_cross_entropy(x, w, target), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), x)


def test_gradients_of_a_gradient_that_is_followed_are_refused():
    x, w, target = _inputs(20, 50, 16, "f32")
    loss = table_cross_entropy(x, w, target)
    g = torch.ones_like(loss).requires_grad_()
    d, = torch.autograd.grad(loss, x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        d.sum().backward()


def test_saved_tensors_elsewhere():
    """Hooks that move what is saved to the host and back."""
    x, w, target = _inputs(90, 200, 40, "bf16", 0.2)
    want = torch.autograd.grad(table_cross_entropy(x, w, target), (x, w))
    with torch.autograd.graph.save_on_cpu():
        loss = table_cross_entropy(x, w, target)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w)), want))


def test_table_of_more_than_4_gib():
    """Entries whose offsets pass 32 bits, with two rows that belong to the last ones; the oracle in pieces, in double precision."""
    t, c = 280_000, 8192
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.empty(t, c, dtype=torch.bfloat16, device="cuda").normal_(0, 2 / c ** 0.5, generator=g).requires_grad_()
    target = torch.tensor([t - 1, 5, -1, t - 2], device="cuda")
    x = (torch.randn(4, c, device="cuda", generator=g) + 1.5 * w.detach()[target].float()).bfloat16().requires_grad_()
    loss = table_cross_entropy(x, w, target, reduction="none")
    d_rows, d_table = torch.autograd.grad(loss, (x, w), torch.ones(4, device="cuda"))
    rows = x.detach()[[0, 1, 3]].double()
    logits = torch.cat([rows @ part.double().t() for part in w.detach().split(20_000)], 1)
    p = torch.log_softmax(logits, 1)
    own = target[[0, 1, 3]]
    assert (loss[[0, 1, 3]].double() + p[[0, 1, 2], own]).abs().max() < 1e-3 and float(loss[2].detach()) == 0
    p = p.exp_()
    p[[0, 1, 2], own] -= 1
    for first in (0, 262_144 - 64, t - 128):  # (2^32 bytes are 262,144 entries)
        part = slice(first, first + 128)
        want, size = p[:, part].t() @ rows, p[:, part].abs().t() @ rows.abs()
        assert ((d_table[part].double() - want).abs() <= 2.0 ** -7 * size + 1e-6).all()
    want = sum(p[:, i:i + 20_000] @ w.detach()[i:i + 20_000].double() for i in range(0, t, 20_000))
    size = sum(p[:, i:i + 20_000].abs() @ w.detach()[i:i + 20_000].double().abs() for i in range(0, t, 20_000))
    assert ((d_rows[[0, 1, 3]].double() - want).abs() <= 2.0 ** -7 * size + 1e-6).all() and (d_rows[2] == 0).all()


def test_refusals():
    x, w, target = _inputs(20, 50, 16, "f32")
    for args, message in (((x, w[:, :8], target), "channels"), ((x, w.bfloat16(), target), "one type"), ((x, w, target[:5]), "target"),
                          ((x, w, target.float()), "int32 or int64"), ((x[0], w, target), "rows"), ((x, w[0], target), "table"),
                          ((x.cpu(), w, target), "rows"), ((x, w.cpu(), target), "table"), ((x.double(), w.double(), target), "rows")):
        with pytest.raises((ValueError, RuntimeError), match=message):
            table_cross_entropy(*args)
    with pytest.raises(RuntimeError, match="GPU"):
        table_cross_entropy(x, w, target.cpu())
    with pytest.raises(ValueError, match="reduction"):
        table_cross_entropy(x, w, target, reduction="median")
    with pytest.raises(RuntimeError, match="scale"):
        table_cross_entropy(x, w, target, scale=float("nan"))
    with pytest.raises(RuntimeError, match="num_channels"):
        table_cross_entropy(x[:, :0], w[:, :0], target)
