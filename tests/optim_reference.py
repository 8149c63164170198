"""AdamW and its 8-bit moments in double precision with numpy, written from the formulas of include/trips_optim.h."""
import numpy as np

BLOCK = 256


def fp8_values(mantissa, bias, codes):
    """The numbers that codes of an 8-bit float stand for (finite ones)."""
    codes = np.asarray(codes, dtype=np.int64)
    sign = np.where(codes & 0x80, -1.0, 1.0)
    e = (codes & 0x7F) >> mantissa
    f = (codes & ((1 << mantissa) - 1)) / float(1 << mantissa)
    return sign * np.where(e == 0, f * 2.0 ** (1 - bias), (1 + f) * 2.0 ** (e - bias))


def mix(x):
    x = np.asarray(x, dtype=np.uint64) & np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(16)
    x = x * np.uint64(0x9E3779B9) & np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(15)
    x = x * np.uint64(0xB504F333) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def encode(x, r, mantissa, bias, largest, positive):
    """(codes, scales, distance of the nearest border in steps): x in blocks, rounded with the 16-bit numbers r."""
    n = x.size
    blocks = -(-n // BLOCK)
    wide = np.zeros(blocks * BLOCK)
    wide[:n] = np.where(np.isfinite(x), np.abs(x), 0.0)
    top = wide.reshape(blocks, BLOCK).max(axis=1)
    k = np.full(blocks, -118)
    for b in np.nonzero(top)[0]:
        k[b] = -118
        while k[b] < 111 and top[b] > largest * 2.0 ** k[b]:
            k[b] += 1
    grid = np.unique(np.abs(fp8_values(mantissa, bias, np.arange(0x80))))
    grid = grid[grid <= largest]
    finite = np.isfinite(x)
    y = np.abs(np.where(finite, x, 0.0)) / 2.0 ** k[np.arange(n) // BLOCK]
    low = np.clip(np.searchsorted(grid, y, side="right") - 1, 0, grid.size - 1)
    high = np.minimum(low + 1, grid.size - 1)
    part = np.where(high > low, (y - grid[low]) / np.where(high > low, grid[high] - grid[low], 1.0), 0.0)
    at = part + (r + 0.5) / 65536.0
    code = np.where(at >= 1.0, high, low)  # (the grid is in the order of the codes)
    if positive:
        code = np.where((x > 0) & (code == 0), 1, code)
    code = np.where(finite, code, 0x7F)
    code = code | np.where(np.signbit(x), 0x80, 0)
    return code.astype(np.uint8), 2.0 ** k, np.abs(at - 1.0)[finite].min() if finite.any() else 1.0


def decode(codes, scales, mantissa, bias):
    return fp8_values(mantissa, bias, codes) * np.asarray(scales, dtype=np.float64)[np.arange(np.size(codes)) // BLOCK]


def step(w, g, m, v, t, lr, betas, eps, decay, factor=1.0):
    """(w, m, v) after step t, and the size of the update's terms (for error bounds); all in double."""
    b1, b2 = betas
    g = g.astype(np.float64) * factor
    m2 = b1 * m + (1 - b1) * g
    v2 = b2 * v + (1 - b2) * g * g
    with np.errstate(invalid="ignore", divide="ignore"):
        denominator = np.sqrt(v2) / np.sqrt(1 - b2 ** t) + eps
        update = lr / (1 - b1 ** t) * m2 / denominator
        terms = lr / (1 - b1 ** t) * (b1 * np.abs(m) + (1 - b1) * np.abs(g)) / denominator
    return w * (1 - lr * decay) - update, m2, v2, terms
