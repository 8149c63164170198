"""Rows and tables whose gradients are 0 as sums of numbers that are not, so that half a step of 16 bits in one of those shows; the bound of d_ij held in two parts of 16 bits."""
import numpy as np
import torch

U = 2.0 ** -24  # half a step of float32, relative to the value
# (the tiles of 64 and the few rows that two parts are for)
SIZES = [(1, 300, 8), (9, 19, 100), (30, 900, 40), (120, 5000, 64), (300, 1000, 100), (900, 333, 33), (700, 150, 16), (129, 4000, 24)]


def zero_for_rows(n, t, c, dtype, device="cpu"):
    """The first channel is the same in all entries: its gradient of a row is that times the sum of the row's d_ij, which is 0."""
    rng = np.random.default_rng(n + t + c)
    x, w = rng.normal(size=(n, c)), rng.normal(size=(t, c)) / np.sqrt(c)
    w[:, 0] = 1
    return (*(torch.as_tensor(a).to(dtype).to(device) for a in (x, w)), torch.as_tensor(rng.integers(0, t, n), device=device), torch.ones(n, device=device))


def zero_for_the_table(n, t, c, dtype, device="cpu"):
    """Rows come in threes that are alike, with gradients of 1, 2 and -3 of their losses."""
    x, w, target, _ = zero_for_rows(n, t, c, dtype, device)
    return x.repeat(3, 1), w, target.repeat(3), torch.tensor([1.0, 2.0, -3.0], device=device).repeat_interleave(n)


def d(x, w, target, weights):
    """d_ij in double precision."""
    p = torch.softmax(x.double() @ w.double().t(), 1)
    p[torch.arange(x.shape[0], device=x.device), target] -= 1
    return p * weights.double()[:, None]


def bound(x, w, weights, sizes, terms):
    """Of a sum of `terms` d_ij times numbers, whose sizes add up to `sizes`: d_ij is held to half a step of half a step, a probability is off by that of its
    exponent (2 U of logits up to 64) and of its exponential and logarithm (32 U); additions by up to 2 U each, independent of one another, so 8 standard deviations of them 16 U times
    the root of their number; float16's smallest step is 2^-24 / 32768 of the largest gradient. Half a step of a result that small is half a step of the bound."""
    step = torch.finfo(x.dtype).eps / 2
    assert float((x.double() @ w.double().t()).abs().max()) < 64
    of = (step * step + (2 * 64 + 32 + 16 * terms ** 0.5) * U) * sizes
    low = 2.0 ** -25 / 32768 * float(weights.abs().max()) * terms * float(max(x.abs().max(), w.abs().max())) if x.dtype is torch.float16 else 0.0
    return (of + low) * (1 + step) + torch.finfo(x.dtype).smallest_normal * step
