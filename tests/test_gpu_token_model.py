"""A small model over a table's rows as a program trains it: rows looked up by token, dropped out, through a layer, scored against the same table, both
ends' gradients, clipping and an AdamW step; against the same step in torch's own operations in double precision, eagerly and captured."""
import numpy as np
import pytest
import torch

from tests.loss_reference import kept
from trips_amd.adamw import AdamW
from trips_amd.dropout import dropout
from trips_amd.lookup import ROWS, lookup
from trips_amd.table_loss import table_cross_entropy

pytestmark = pytest.mark.gpu
SEED, P, LR = 77, 0.25, 1e-2


def _model(dtype, entries=300, channels=48, tokens=190):
    g = torch.Generator(device="cuda").manual_seed(4)
    table = torch.nn.Parameter((torch.randn(entries, channels, device="cuda", generator=g) * 0.3).to(dtype))
    weight = torch.nn.Parameter((torch.randn(channels, channels, device="cuda", generator=g) / channels ** 0.5).to(dtype))
    token = torch.randint(0, entries, (tokens,), device="cuda", generator=g)
    target = torch.roll(token, -1)
    token[::17], target[::11] = -1, -1
    return table, weight, token, target


def _loss(table, weight, token, target, step):
    rows = lookup(table, token, scale=2.0, layout=ROWS)
    out = dropout(rows @ weight, P, SEED, call=1, step=step, residual=dropout(rows, P, SEED, call=0, step=step))
    return table_cross_entropy(out, table, target, scale=0.8)


def _expected(table, weight, token, target, step, rounded):
    """The loss and its gradients in double precision; `rounded` is what each operator's result goes through."""
    t, w = (p.detach().double().cpu().requires_grad_() for p in (table, weight))
    token, target = token.cpu(), target.cpu()
    inside = token >= 0
    rows = rounded(torch.where(inside[:, None], t[token.clamp(min=0)] * 2.0, torch.zeros((), dtype=torch.float64)))

    def drop(x, call):
        keep, factor = kept(x.numel(), P, SEED, call, step)
        return x * torch.as_tensor(keep.reshape(x.shape) * factor)
    out = rounded(drop(rounded(rows @ w), 1) + rounded(drop(rows, 0)))
    counted = target >= 0
    loss = torch.nn.functional.cross_entropy(0.8 * out[counted] @ t.t(), target[counted])
    return (loss, *torch.autograd.grad(loss, (t, w)))


class _Rounded(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dtype):
        return x.to(dtype).double()

    @staticmethod
    def backward(ctx, g):
        return g, None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_of_the_whole(dtype):
    """Every operator's result and every gradient that one hands on is rounded to the type once (half a step, five of them on a way at most, and the
    sum of the table's two ends): 6 half steps of the gradients' root mean square, and of single elements 40."""
    model = _model(dtype)
    step = torch.full((), 9, dtype=torch.int32, device="cuda")
    loss = _loss(*model, step)
    got = (loss, *torch.autograd.grad(loss, model[:2]))
    want = _expected(*model, 9, lambda x: _Rounded.apply(x, dtype))
    half = torch.finfo(dtype).eps / 2
    assert abs(float(got[0].detach()) - float(want[0].detach())) <= 6 * half * float(want[0].detach())
    for a, b in zip(got[1:], want[1:]):
        err, size = (a.double().cpu() - b), float(b.square().mean().sqrt())
        assert float(err.square().mean().sqrt()) <= 6 * half * size + 1e-6 * size
        assert float(err.abs().max()) <= 40 * half * (size + float(b.abs().max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_training_is_the_eager_one(dtype):
    """Steps from a graph, whose dropout follows the optimiser's own step count on the device, and the same steps without one: the same bits."""
    weights = []
    for captured in (False, True):
        table, weight, token, target = _model(dtype)
        opt = AdamW([table, weight], lr=LR, max_grad_norm=1.0, min_8bit_size=0, state_bits=8, seed=SEED)

        def step(count):
            table.grad, weight.grad = torch.autograd.grad(_loss(table, weight, token, target, count), (table, weight))
            opt.step()
        zero = torch.zeros((), dtype=torch.int32, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(zero)  # (a first step makes the state)
        torch.cuda.synchronize()
        count = opt.state[table]["step"]
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(count)
        seen = []
        for i in range(4):
            if captured:
                graph.replay()
            else:
                with torch.cuda.stream(side):
                    step(count)
            torch.cuda.synchronize()
            assert int(count) == i + 2
            seen.append((table.detach().clone(), weight.detach().clone()))
        weights.append(seen)
    for a, b in zip(*weights):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(weights[0][0][0], weights[0][3][0])


def test_single_tokens_are_scored_as_in_a_batch():
    """What a row loses by itself, as an answer is scored token by token, within the bound of a batch's (in other tiles, the same products)."""
    table, _, token, target = _model(torch.bfloat16, entries=5000, channels=256, tokens=300)
    with torch.no_grad():
        rows = lookup(table, token, layout=ROWS)
        together = table_cross_entropy(rows, table, target, reduction="none")
        for i in (0, 1, 18, 150, 299):
            alone = table_cross_entropy(rows[i:i + 1], table, target[i:i + 1], reduction="none")
            size = float((rows[i].double().abs() @ table.double().abs().t()).max())
            assert abs(float(alone) - float(together[i])) <= 2.0 ** -23 * (258 * 4 * size + 800)
    assert float(together[target < 0].abs().sum()) == 0


def test_on_another_device_index():
    """All of it names the device of its tensors; one that is not there is torch's to refuse."""
    table, weight, token, target = _model(torch.float32)
    with torch.cuda.device(0):
        loss = _loss(table.to("cuda:0"), weight, token, target, 3)
    assert np.isfinite(float(loss.detach()))
