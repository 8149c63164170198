"""Plain forms in double precision of a table's cross entropy and of dropout, and the bounds that the kernels' results are held to."""
import numpy as np
import torch

U = 2.0 ** -24  # half a step of float32, relative to the value


def half_step(dtype, value):
    """What rounding to `dtype` (through float32) takes at most."""
    if dtype is torch.float32:
        return np.abs(value) * U + 2.0 ** -149
    info = torch.finfo(dtype)
    return np.abs(value) * (info.eps / 2 * (1 + 4 * U) + U) + info.smallest_normal * info.eps / 2


def philox(counter, key):
    """Philox-4x32-10 of counters [n, 4] and a key of two words: [n, 4], all in uint64 arrays that hold 32 bits."""
    c = [np.array(counter[:, i], dtype=np.uint64) for i in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    mask, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ np.uint64(k0), b & mask, (a >> shift) ^ c[3] ^ np.uint64(k1), a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1)


def kept(n, p, seed, call, step, first=0):
    """Which of the elements first .. first + n - 1 (first a multiple of 8) are kept, and the factor of those."""
    blocks = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    counter = np.stack([blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32), np.full_like(blocks, call), np.full_like(blocks, step & 0xFFFFFFFF)], 1)
    words = philox(counter, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)[:n]
    border = int(np.round(p * 65536))  # (ties to even)
    return halves >= border, 65536.0 / (65536 - border) if border < 65536 else 0.0


class Loss:
    """The cross entropy of rows against a table, in double precision, and how far the kernels may be off.

    e_i, the products of a row: a sum of C products in float32 in any order, each addition off by at most 2^-23 of the sum of
    magnitudes (the matrix instructions may cut where others round), so C 2^-23 max_j sum_c |x_ic w_jc| |scale|, for C + 2 of them here (two
    more than there are). Both the products and what
    they are compared with are off by e_i; the difference and its scaling add 4 U of their size (at most 2 max_j |l_ij|).
    The exponential is off by 2^-22 of itself, its sum, in chains of at most 320 + T / 64 terms, by as many U."""

    def __init__(self, rows, table, target, scale, weights):
        """weights [N]: the gradient of each row's loss, zero where a row does not count."""
        self.dtype = rows.dtype
        x, w = rows.detach().double().cpu().numpy(), table.detach().double().cpu().numpy()
        t = target.detach().cpu().numpy().reshape(-1).astype(np.int64)
        self.counts = (t >= 0) & (t < w.shape[0])
        self.losses, self.d_rows = np.zeros(x.shape[0]), np.zeros_like(x)
        self.d_table = np.zeros_like(w)
        scale = float(np.float32(scale))
        i = np.nonzero(self.counts)[0]
        n, channels = i.size, x.shape[1]
        self.loss_bound, self.d_rows_bound, self.d_table_bound = np.zeros(x.shape[0]), half_step(self.dtype, self.d_rows), half_step(self.dtype, self.d_table)
        if n == 0:
            return
        x, t, g = x[i], t[i], np.asarray(weights, dtype=np.float64)[i]
        l = scale * (x @ w.T)
        top = l.max(1, keepdims=True)
        e = np.exp(l - top)
        total = e.sum(1, keepdims=True)
        p = e / total
        at = np.arange(n)
        self.losses[i] = np.log(total[:, 0]) + top[:, 0] - l[at, t]
        d = p.copy()
        d[at, t] -= 1
        d *= g[:, None]
        self.d_rows[i], self.d_table = scale * (d @ w), scale * (d.T @ x)
        # bounds
        size = abs(scale) * (np.abs(x) @ np.abs(w).T).max(1)
        terms = channels + 2
        off = 2 * terms * 2 * U * size + 8 * U * np.abs(l).max(1) + (320 + w.shape[0] / 64 + 8) * U  # of a log probability
        self.loss_bound[i] = off + 4 * U * np.abs(self.losses[i])
        u_d = U if self.dtype is torch.float32 else torch.finfo(self.dtype).eps / 2
        low = 0.0
        if self.dtype is torch.float16:  # (held 2^15 / max |g| times as large, smallest step 2^-24)
            low = 2.0 ** -25 * np.abs(g).max() / 32768
        d_off = np.abs(g)[:, None] * p * np.expm1(2 * off)[:, None] + np.abs(d) * (u_d + 8 * U) + 2 * U * np.abs(g)[:, None] * p + low
        d_off[at, t] += 4 * U * np.abs(g)
        s = abs(scale)
        self.d_rows_bound[i] = s * (d_off @ np.abs(w) + (w.shape[0] + 8) * 2 * U * (np.abs(d) @ np.abs(w))) + half_step(self.dtype, self.d_rows[i])
        self.d_table_bound = s * (d_off.T @ np.abs(x) + (n + 8) * 2 * U * (np.abs(d).T @ np.abs(x))) + half_step(self.dtype, self.d_table)


def within(got, want, bound, what):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = np.abs(got - want)
    ok = err <= bound  # (false for NaN)
    assert ok.all(), f"{what}: {(~ok).sum()} of {ok.size} off, {np.nanmax(err / np.maximum(bound, 1e-300)):.3g} times the bound, first at {np.argwhere(~ok)[0]}"
