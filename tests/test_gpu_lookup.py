"""Lookups, the order of their points and their gradient, against numpy in double precision.

Bounds: a lookup is one product in float32 (2^-24 of it) and one rounding to its type (half a step); a sum of k terms in
float32, in any order, is off by at most k 2^-24 of the sum of their magnitudes, its scaling and rounding as the lookup's."""
import numpy as np
import pytest
import torch

from trips_amd import lookup as lk

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BOTH = [lk.COLUMNS, lk.ROWS]


def _numbers(t):
    return t.detach().double().cpu().numpy()


def _half_step(dtype, value):
    if dtype is torch.float32:
        return np.abs(value) * U
    info = torch.finfo(dtype)
    return np.abs(value) * (info.eps / 2 * (1 + 4 * U) + U) + info.smallest_normal * info.eps / 2


def _index(rng, texels, points, how, dtype=torch.int32):
    if how == "same":
        i = np.full(points, texels // 2)
    elif how == "skewed":
        i = (texels * rng.random(points) ** 4).astype(np.int64)
    elif how == "outside":
        i = rng.integers(-2, texels + 2, points)
    elif how == "all_outside":
        i = np.full(points, -1)
    elif how == "once":
        i = rng.permutation(max(texels, points))[:points]
    else:
        i = rng.integers(0, max(texels, 1), points)
    return torch.as_tensor(i, dtype=dtype, device="cuda")


def _matrix(rng, rows, columns, dtype, pad=0, spread=0.0):
    """A matrix whose rows lie `pad` elements apart."""
    x = rng.normal(size=(rows, columns + pad)) * np.exp(spread * rng.normal(size=(rows, columns + pad)))
    return torch.as_tensor(x, dtype=TYPES[dtype], device="cuda")[:, :columns]


def _inside(index, texels):
    i = index.cpu().numpy().astype(np.int64).reshape(-1)
    return i, (i >= 0) & (i < texels)


def _check_lookup(got, table, index, scale, layout):
    t = _numbers(table) if layout == lk.ROWS else _numbers(table).T
    i, ok = _inside(index, t.shape[0])
    want = np.zeros((i.size, t.shape[1]))
    want[ok] = t[i[ok]] * np.float64(np.float32(scale))
    out = _numbers(got) if layout == lk.ROWS else _numbers(got).T
    assert out.shape == want.shape
    assert (np.abs(out - want) <= U * np.abs(want) + _half_step(table.dtype, want)).all()
    assert (out[~ok] == 0).all()


def _check_grad(got, grad, index, texels, scale, layout, before=None):
    g = _numbers(grad) if layout == lk.ROWS else _numbers(grad).T
    i, ok = _inside(index, texels)
    want, size = np.zeros((texels, g.shape[1])), np.zeros((texels, g.shape[1]))
    np.add.at(want, i[ok], g[ok])
    np.add.at(size, i[ok], np.abs(g[ok]))
    k = np.bincount(i[ok], minlength=texels)[:, None]
    s = np.float64(np.float32(scale))
    want, size = want * s, size * abs(s)
    extra = 0.0
    if before is not None:
        b = _numbers(before) if layout == lk.ROWS else _numbers(before).T
        want = want + b
        extra = U * np.abs(want)
    out = _numbers(got) if layout == lk.ROWS else _numbers(got).T
    assert out.shape == want.shape
    bound = (k + 2) * U * size + _half_step(grad.dtype, want) + extra
    err = np.abs(out - want)
    assert (err <= bound).all(), (err / np.maximum(bound, 1e-300)).max()
    if before is None:
        assert (out[k[:, 0] == 0] == 0).all()


def _check_plan(plan, index, texels):
    i, ok = _inside(index, texels)
    key = np.where(ok, i, texels)
    np.testing.assert_array_equal(plan.order.cpu().numpy(), np.argsort(key, kind="stable"))
    np.testing.assert_array_equal(plan.starts.cpu().numpy(), np.searchsorted(np.sort(key), np.arange(texels + 1)))


PLANS = [(1, 1, "any"), (1, 5000, "same"), (2, 1, "any"), (7, 64, "outside"), (255, 4095, "any"), (256, 4096, "any"), (257, 4097, "outside"),
         (300, 100_000, "skewed"), (65_535, 70_001, "any"), (65_536, 50_000, "outside"), (70_000, 9, "any"), (3_000_000, 20_000, "any"),
         (1 << 24, 300_000, "any"), ((1 << 31) - 100, 1, "none"), (50_000, 300_000, "same"), (1000, 30_000, "all_outside"), (40_000, 40_000, "once"),
         (0, 100, "all_outside"), (100, 0, "any"), (0, 0, "any"), (5000, 16_385, "skewed"), (33, 8192, "outside"), (33, 8193, "outside"),
         (9000, 8191, "any"), (200_000, 8192, "skewed"), (1000, 1_100_000, "skewed"), (2_000_000, 1_200_000, "outside"), (70_000, 65_536, "any"),
         (70_000, 65_537, "any"), (500_000, 1_048_575, "any"), (500_000, 1_048_576, "any"),
         (3_000_000, 4_194_303, "outside"), (3_000_000, 4_194_304, "outside"), (300, 5_000_000, "skewed")]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("texels,points,how", [p for p in PLANS if p[2] != "none"])
def test_plan(texels, points, how, dtype):
    index = _index(np.random.default_rng(texels + points), texels, points, how, dtype)
    _check_plan(lk.lookup_plan(index, texels), index, texels)


@pytest.mark.parametrize("points", [1, 31, 32, 33, 100, 1025])
@pytest.mark.parametrize("texels", [15_359, 15_360, 30_721, 491_519, 491_520, 130_815, 4_194_303, 4_194_304])
def test_plan_of_few_points_and_many_texels(texels, points):
    rng = np.random.default_rng(texels + points)
    index = _index(rng, texels, points, "any")
    index[rng.integers(points)] = texels - 1
    index[rng.integers(points)] = texels
    _check_plan(lk.lookup_plan(index, texels), index, texels)


@pytest.mark.parametrize("how", ["any", "skewed", "outside", "same", "all_outside", "once"])
@pytest.mark.parametrize("points", [1, 63, 64, 65, 1023, 1025, 8192, 8193, 16_385, 24_577, 32_768, 32_769])
@pytest.mark.parametrize("texels", [1, 2, 255, 256, 257, 511, 20_000, 65_535, 245_759, 245_760])
def test_plan_in_one_launch(texels, points, how):
    """About the sizes at which the kernel, its rounds or the texels of a workgroup change."""
    index = _index(np.random.default_rng(texels + 3 * points), texels, points, how, torch.int64 if points % 2 else torch.int32)
    _check_plan(lk.lookup_plan(index, texels), index, texels)


def test_plan_of_indexes_beyond_32_bits():
    index = torch.tensor([1 << 32, 5, -(1 << 40), (1 << 31) + 5, 0, 5], device="cuda")
    plan = lk.lookup_plan(index, 6)
    _check_plan(plan, index, 6)
    assert plan.starts[-1] == 3


LOOKS = [(1, 1, 1), (1, 300, 3), (7, 1, 4), (100, 257, 5), (1000, 4097, 16), (33, 1000, 17), (50, 129, 64), (1000, 513, 200), (300, 100, 1024),
         (40, 70, 1031), (5, 9, 4100)]


@pytest.mark.parametrize("layout", BOTH)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("texels,points,channels", LOOKS)
@pytest.mark.parametrize("pad", [0, 3])
def test_lookup_and_gradient(texels, points, channels, dtype, layout, pad):
    rng = np.random.default_rng(texels * 7 + points + channels)
    for how, index_dtype, scale in (("outside", torch.int32, 1.0), ("skewed", torch.int64, -2.7)):
        index = _index(rng, texels, points, how, index_dtype)
        rows, columns = (texels, channels) if layout == lk.ROWS else (channels, texels)
        table = _matrix(rng, rows, columns, dtype, pad)
        _check_lookup(lk.lookup(table, index, scale, layout), table, index, scale, layout)
        rows, columns = (points, channels) if layout == lk.ROWS else (channels, points)
        grad = _matrix(rng, rows, columns, dtype, pad, spread=1.0)
        got = lk.lookup_backward(grad, index, texels, scale, layout)
        _check_grad(got, grad, index, texels, scale, layout)
        plan = lk.lookup_plan(index, texels)
        assert torch.equal(lk.lookup_backward(grad, index, texels, scale, layout, plan), got)
        # added to what is there, in a matrix with a gap between its rows
        rows, columns = (texels, channels) if layout == lk.ROWS else (channels, texels)
        wide = _matrix(rng, rows, columns + pad, dtype)
        before = wide.clone()
        out = lk.lookup_backward(grad, index, texels, scale, layout, plan, out=wide[:, :columns])
        _check_grad(out, grad, index, texels, scale, layout, before[:, :columns])
        assert torch.equal(wide[:, columns:], before[:, columns:])


@pytest.mark.parametrize("layout", BOTH)
@pytest.mark.parametrize("channels", [1, 2, 7, 40, 256, 2100])
@pytest.mark.parametrize("texels,how", [(1, "same"), (4, "any"), (9, "outside"), (40, "skewed"), (5000, "skewed")])
@pytest.mark.parametrize("points", [32, 33, 64, 65, 255, 256, 257, 512, 513])
def test_gradient_of_few_points(points, texels, how, channels, layout):
    """Several texels with many of the points, in one workgroup and in several."""
    rng = np.random.default_rng(points * 11 + texels + channels)
    index = _index(rng, texels, points, how)
    for dtype in ("f32", "f16"):
        rows, columns = (points, channels) if layout == lk.ROWS else (channels, points)
        grad = _matrix(rng, rows, columns, dtype, spread=1.0)
        got = lk.lookup_backward(grad, index, texels, 1.5, layout)
        _check_grad(got, grad, index, texels, 1.5, layout)
        rows, columns = (texels, channels) if layout == lk.ROWS else (channels, texels)
        out = _matrix(rng, rows, columns, dtype)
        before = out.clone()
        lk.lookup_backward(grad, index, texels, 1.5, layout, lk.lookup_plan(index, texels), out=out)
        _check_grad(out, grad, index, texels, 1.5, layout, before)


LONG = [(1, 100_000, "same"), (3, 50_000, "any"), (1000, 200_000, "skewed"), (5, 2047, "any"), (2, 2048, "same"), (2, 2049, "same"), (2, 4097, "any"),
        (4000, 300_000, "any"), (1, 130, "same"), (64, 9000, "outside"), (65, 70_000, "skewed")]


@pytest.mark.parametrize("layout", BOTH)
@pytest.mark.parametrize("channels", [1, 4, 6, 40, 300])
@pytest.mark.parametrize("texels,points,how", LONG)
def test_gradient_of_entries_with_many_points(texels, points, how, channels, layout):
    """Sums of thousands of terms; the same bits every time."""
    rng = np.random.default_rng(points + channels)
    if channels == 300:
        points = points // 4 + 1
    index = _index(rng, texels, points, how)
    for dtype in ("f32", "bf16"):
        rows, columns = (points, channels) if layout == lk.ROWS else (channels, points)
        grad = _matrix(rng, rows, columns, dtype)
        got = lk.lookup_backward(grad, index, texels, 0.5, layout)
        _check_grad(got, grad, index, texels, 0.5, layout)
        assert torch.equal(lk.lookup_backward(grad, index, texels, 0.5, layout), got)


@pytest.mark.parametrize("layout", BOTH)
def test_empty_tables_and_no_points(layout):
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    some = torch.zeros(5, dtype=torch.int32, device="cuda")
    for texels, index in ((0, none), (0, some), (4, none)):
        n = index.numel()
        table = torch.ones((texels, 3) if layout == lk.ROWS else (3, texels), device="cuda")
        got = lk.lookup(table, index, layout=layout)
        assert got.shape == ((n, 3) if layout == lk.ROWS else (3, n)) and not got.any()
        got = lk.lookup_backward(torch.ones_like(got), index, texels, layout=layout)
        assert got.shape == table.shape and not got.any()


@pytest.mark.parametrize("layout", BOTH)
def test_infinities_stay_with_their_entry(layout):
    index = torch.tensor([0, 2, 2, 3, -1], dtype=torch.int32, device="cuda")
    grad = torch.ones((5, 4), device="cuda")
    grad[1, 0], grad[3, 1], grad[4] = float("inf"), float("nan"), float("inf")
    got = lk.lookup_backward(grad if layout == lk.ROWS else grad.t().contiguous(), index, 5, layout=layout)
    got = (got if layout == lk.ROWS else got.t()).cpu().numpy()
    want = np.array([[1, 1, 1, 1], [0, 0, 0, 0], [np.inf, 2, 2, 2], [1, np.nan, 1, 1], [0, 0, 0, 0]])
    np.testing.assert_array_equal(got, want)
    table = torch.full((2, 4), float("nan"), device="cuda")
    out = lk.lookup(table if layout == lk.ROWS else table.t().contiguous(), torch.tensor([-1, 2], device="cuda"), layout=layout)
    assert not out.any()


@pytest.mark.parametrize("layout", BOTH)
def test_autograd_against_differences(layout):
    """The operator is linear: differences over a step that float32 holds exactly are exact but for the sums' roundings."""
    rng = np.random.default_rng(5)
    index = _index(rng, 6, 40, "outside")
    table = _matrix(rng, *((6, 3) if layout == lk.ROWS else (3, 6)), "f32").contiguous().requires_grad_()
    weights = torch.randn((40, 3) if layout == lk.ROWS else (3, 40), device="cuda")
    plan = lk.lookup_plan(index, 6)
    for p in (None, plan):
        table.grad = None
        (lk.lookup(table, index, 1.5, layout, p) * weights).sum().backward()
        for k in range(18):
            step = torch.zeros(18, device="cuda")
            step[k] = 1.0
            step = step.reshape(table.shape)
            with torch.no_grad():
                up, down = (lk.lookup(table + s * step, index, 1.5, layout).double() for s in (1, -1))
                slope = float(((up - down) * weights.double()).sum() / 2)
            assert abs(float(table.grad.reshape(-1)[k]) - slope) <= 1e-5 * float(weights.abs().sum())
    # a broadcast table: its gradient is summed over what it was broadcast from
    row = torch.randn(1, 3, device="cuda", requires_grad=True)
    (lk.lookup(row.expand(6, 3), index, 1.0, lk.ROWS)).sum().backward()
    inside = int(((index >= 0) & (index < 6)).sum())
    assert torch.equal(row.grad, torch.full((1, 3), float(inside), device="cuda"))
    # a gradient that is a broadcast number
    table.grad = None
    lk.lookup(table, index, 1.0, layout).sum().backward()
    counts = torch.bincount(index[(index >= 0) & (index < 6)].long(), minlength=6).float()
    assert torch.equal(table.grad, (counts[:, None] if layout == lk.ROWS else counts[None]).expand_as(table))


def test_index_of_other_strides_and_shapes():
    rng = np.random.default_rng(6)
    wide = _index(rng, 50, 400, "outside").reshape(200, 2)
    index = wide[:, 0]
    table = _matrix(rng, 4, 50, "f32")
    got = lk.lookup(table, index)
    _check_lookup(got, table, index, 1.0, lk.COLUMNS)
    plan = lk.lookup_plan(index, 50)
    _check_plan(plan, index.contiguous(), 50)
    grad = _matrix(rng, 200, 4, "f32").t()  # its rows are not rows of memory
    _check_grad(lk.lookup_backward(grad, index, 50, plan=plan), grad, index, 50, 1.0, lk.COLUMNS)
    column = wide[:, :1].contiguous()  # [N, 1], as a scene keeps it
    assert torch.equal(lk.lookup(table, column), got)


def test_plans_of_other_indexes_are_refused():
    index = torch.tensor([1, 2, 0, 1], dtype=torch.int32, device="cuda")
    plan = lk.lookup_plan(index, 3)
    grad = torch.ones(2, 4, device="cuda")
    with pytest.raises(ValueError, match="plan"):
        lk.lookup_backward(grad, index.clone(), 3, plan=plan)
    with pytest.raises(ValueError, match="plan"):
        lk.lookup_backward(grad, index, 4, plan=plan)
    index[0] = 2
    with pytest.raises(ValueError, match="changed"):
        lk.lookup_backward(grad, index, 3, plan=plan)
    own = lk.LookupPlan(plan.order, plan.starts)  # a program's own tensors are taken at their word
    lk.lookup_backward(grad, index, 3, plan=own)
    table = torch.ones(2, 3, device="cuda", requires_grad=True)
    out = lk.lookup(table, index)
    index[0] = 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("layout", BOTH)
def test_a_plan_with_wild_numbers_stays_inside(layout):
    """Points and starts that lie outside are passed over, not followed."""
    n, t = 3000, 7
    index = torch.arange(n, dtype=torch.int32, device="cuda") % t
    good = lk.lookup_plan(index, t)
    order, starts = good.order.clone(), good.starts.clone()
    order[::3] = -5
    order[1::3] = 2 ** 31 - 1
    starts[2] = 2 ** 31 - 1
    starts[4] = -7
    grad = torch.ones((n, 4) if layout == lk.ROWS else (4, n), device="cuda")
    got = lk.lookup_backward(grad, index, t, layout=layout, plan=lk.LookupPlan(order, starts))
    assert torch.isfinite(got).all() and float(got.max()) <= n


@pytest.mark.parametrize("layout", BOTH)
@pytest.mark.parametrize("points", [40, 400, 5000])
def test_a_plan_in_which_every_other_texel_has_all_points(points, layout):
    """More long texels than a sound plan can have: those that find no room are left out, nothing else happens."""
    t = 3000
    order = torch.arange(points, dtype=torch.int32, device="cuda")
    starts = torch.where(torch.arange(t + 1, device="cuda") % 2 == 0, 0, points).to(torch.int32)
    for channels in (1, 4):
        grad = torch.ones((points, channels) if layout == lk.ROWS else (channels, points), device="cuda")
        index = torch.zeros(points, dtype=torch.int32, device="cuda")
        out = torch.zeros((t, channels) if layout == lk.ROWS else (channels, t), device="cuda")
        lk.lookup_backward(grad, index, t, layout=layout, plan=lk.LookupPlan(order, starts), out=out)
        rows = out if layout == lk.ROWS else out.t()
        assert (rows[1::2] == 0).all()
        assert ((rows[::2] == points) | (rows[::2] == 0)).all()


def test_refusals():
    index = torch.zeros(4, dtype=torch.int32, device="cuda")
    table = torch.zeros(3, 5, device="cuda")
    for bad in (table.double(), table.int(), table.cpu(), table[0]):
        with pytest.raises(ValueError):
            lk.lookup(bad, index)
    with pytest.raises(ValueError):
        lk.lookup(table, index.float())
    with pytest.raises(ValueError, match="points"):
        lk.lookup_backward(torch.zeros(3, 5, device="cuda"), index, 5)
    with pytest.raises(ValueError):
        lk.lookup_plan(index, -1)
    grad = torch.zeros(3, 4, device="cuda")
    for out in (torch.zeros(3, 6, device="cuda"), torch.zeros(3, 5, device="cuda", dtype=torch.bfloat16), torch.zeros(5, 3, device="cuda").t(),
                torch.zeros(1, 5, device="cuda").expand(3, 5)):
        with pytest.raises(ValueError, match="out"):
            lk.lookup_backward(grad, index, 5, out=out)
    with pytest.raises(ValueError, match="int32"):
        lk.LookupPlan(torch.zeros(4, device="cuda"), torch.zeros(6, device="cuda"))


@pytest.mark.parametrize("layout", BOTH)
def test_captured_lookup_and_gradient_replay(layout):
    """New indexes, tables and gradients in the same memory before every replay; eager work in between."""
    rng = np.random.default_rng(8)
    texels, points, channels = 700, 20_000, 4
    index = _index(rng, texels, points, "skewed")
    table = _matrix(rng, *((texels, channels) if layout == lk.ROWS else (channels, texels)), "f32").contiguous()
    grad = _matrix(rng, *((points, channels) if layout == lk.ROWS else (channels, points)), "f32").contiguous()
    lk.lookup_backward(grad, index, texels, 2.0, layout)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        values = lk.lookup(table, index, 2.0, layout)
        d_table = lk.lookup_backward(grad, index, texels, 2.0, layout)
    for k in range(4):
        index.copy_(_index(rng, texels, points, ("skewed", "same", "outside", "any")[k]))
        table.normal_()
        grad.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(values, lk.lookup(table, index, 2.0, layout))
        assert torch.equal(d_table, lk.lookup_backward(grad, index, texels, 2.0, layout))
        _check_grad(d_table, grad, index, texels, 2.0, layout)
        torch.randn(50_000, device="cuda").sort()
        torch.cuda.synchronize()


@pytest.mark.parametrize("layout", BOTH)
@pytest.mark.parametrize("texels,points,channels", [(30, 300, 4), (9000, 7000, 1), (400_000, 600, 6), (500, 50_000, 5)])
def test_captured_calls_of_other_sizes_replay(texels, points, channels, layout):
    rng = np.random.default_rng(points)
    index = _index(rng, texels, points, "skewed", torch.int64)
    grad = _matrix(rng, *((points, channels) if layout == lk.ROWS else (channels, points)), "bf16").contiguous()
    lk.lookup_backward(grad, index, texels, 1.0, layout)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        plan = lk.lookup_plan(index, texels)
        d_table = lk.lookup_backward(grad, index, texels, 1.0, layout)
    for k in range(3):
        index.copy_(_index(rng, texels, points, ("any", "same", "outside")[k]))
        grad.normal_()
        graph.replay()
        torch.cuda.synchronize()
        _check_plan(plan, index, texels)
        _check_grad(d_table, grad, index, texels, 1.0, layout)
        assert torch.equal(d_table, lk.lookup_backward(grad, index, texels, 1.0, layout))
        torch.randn(50_000, device="cuda").sort()
        torch.cuda.synchronize()


def test_offsets_that_pass_32_bits():
    """Tables and gradients of more than 2^32 elements: their last and first entries."""
    texels = (1 << 22) + 5
    index = torch.tensor([0, texels - 1, 5, texels - 1, texels, texels - 2], dtype=torch.int64, device="cuda")
    table = torch.zeros((texels, 1024), dtype=torch.bfloat16, device="cuda")
    for i in (0, 5, texels - 2, texels - 1):
        table[i] = torch.arange(1024, device="cuda").remainder(13) + i % 7
    got = lk.lookup(table, index, 2.0, lk.ROWS)
    assert torch.equal(got[[0, 1, 2, 3, 5]], table[index[[0, 1, 2, 3, 5]]] * 2) and not got[4].any()
    grad = got.clone()
    del table
    d_table = lk.lookup_backward(grad, index, texels, 1.0, lk.ROWS)
    assert torch.equal(d_table[0], grad[0]) and torch.equal(d_table[5], grad[2]) and torch.equal(d_table[texels - 2], grad[5])
    assert torch.equal(d_table[texels - 1], (grad[1].float() + grad[3].float()).to(torch.bfloat16))
    assert not d_table[6:100].any() and not d_table[texels - 100:texels - 2].any()
    del d_table
    texels = (1 << 30) + 3
    index = torch.tensor([texels - 1, 0, texels - 1, -1, texels, 1 << 29], dtype=torch.int32, device="cuda")
    table = torch.zeros((5, texels), dtype=torch.float16, device="cuda")
    table[:, texels - 1] = torch.arange(1, 6, device="cuda")
    table[:, 0], table[:, 1 << 29] = 7, 9
    got = lk.lookup(table, index, 0.5)
    want = torch.stack([torch.arange(1, 6) * 0.5, torch.full((5,), 3.5), torch.arange(1, 6) * 0.5, torch.zeros(5), torch.zeros(5),
                        torch.full((5,), 4.5)], 1).to(torch.float16).cuda()
    assert torch.equal(got, want)
    del table
    d_table = lk.lookup_backward(want, index, texels, 1.0)
    assert torch.equal(d_table[:, texels - 1], want[:, 0] * 2) and torch.equal(d_table[:, 0], want[:, 1])
    assert torch.equal(d_table[:, 1 << 29], want[:, 5]) and not d_table[:, 1:1000].any() and not d_table[4, texels - 1000:texels - 1].any()


def test_another_stream():
    rng = np.random.default_rng(9)
    index, grad = _index(rng, 500, 60_000, "skewed"), _matrix(rng, 4, 60_000, "f32")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        scaled = grad * 2
        got = lk.lookup_backward(scaled, index, 500)
    side.synchronize()
    _check_grad(got, scaled, index, 500, 1.0, lk.COLUMNS)
