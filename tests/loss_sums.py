"""Gradients of a table that are sums over very many rows: inputs of which every part of the rows is seen in them, the sums in double precision, and a bound that a missing
part falls outside of."""
import torch

U = 2.0 ** -24  # half a step of float32, relative to the value


def inputs(n, t, c, padding, dtype, device, seed=0):
    """Rows without negative numbers, targets among the first half of the entries only: what an entry of the second half gets is a sum without cancellation."""
    g = torch.Generator().manual_seed(seed + n + t + c)
    x = torch.rand(n, c, generator=g).add_(0.25).to(device=device, dtype=dtype)
    w = (torch.randn(t, c, generator=g) / c ** 0.5).to(device=device, dtype=dtype)
    target = (torch.rand(n, generator=g) * ((t + 1) // 2)).long()
    target[torch.rand(n, generator=g) < padding] = -1
    return x, w, target.to(device)


def gradients(x, w, target, weights, leave_out=None):
    """d_rows, d_table and the sums of magnitudes of both, in double precision, a piece of the rows at a time; `leave_out` [N]: rows that a mistake forgets."""
    table, half = w.detach().double(), max(1, 50_000_000 // max(w.shape))
    d_rows, rows_size = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    d_table, table_size = torch.zeros_like(table), torch.zeros_like(table)
    kept = target >= 0 if leave_out is None else (target >= 0) & ~leave_out
    for i in kept.nonzero()[:, 0].split(half):
        rows, at = x.detach()[i].double(), torch.arange(i.numel(), device=x.device)
        d = torch.softmax(rows @ table.t(), 1)
        d[at, target[i]] -= 1
        d *= weights[i].double()[:, None]
        d_rows[i], rows_size[i] = d @ table, d.abs() @ table.abs()
        d_table += d.t().contiguous() @ rows
        table_size += d.abs().t().contiguous() @ rows.abs()
    return d_rows, rows_size, d_table, table_size


def table_bound(x, w, n, d_table, table_size):
    """How far an entry's gradient may be off. Additions in float32 of n terms, in chains that a fixed order joins: each off by at most 2 U (the matrix instructions may cut where others
    round) of a partial sum that is no more than the sum of magnitudes, by themselves independent of one another: 8 standard deviations of n of them, 16 sqrt(n) U of that sum.
    A term is off by what d_ij is: half a step of what holds it in 16 bits, and the error of a probability, whose logits (C products below 1.25 |w|, U of each twice and
    2 U of each addition) enter an exponential. Half a step of the result."""
    c, t = w.shape[1], w.shape[0]
    step = torch.finfo(x.dtype).eps
    logit = (2 * c + 8) * 2 * U * 1.25 * float(w.detach().double().abs().sum(1).max())
    held = 8 * U if x.dtype is torch.float32 else step / 2
    return (16 * n ** 0.5 * U + held + 4 * logit + (320 + t / 64) * U) * table_size + step / 2 * d_table.abs() + 2.0 ** -25
