"""Microscaled 4-bit blocks from their definition: codes, exponents and what they stand for, in float64 numpy."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def blocks(x):
    """(codes [rows, blocks * 32], exponent bytes [rows, blocks]) of the rows of x (float64 array)."""
    rows, cols = x.shape
    nb = -(-cols // 32)
    padded = np.zeros((rows, nb * 32))
    padded[:, :cols] = x
    v = padded.reshape(rows, nb, 32)
    finite = np.isfinite(v).all(2)
    top = np.where(finite, np.abs(np.where(np.isfinite(v), v, 0)).max(2), 0)
    e = np.zeros(top.shape, int)
    e[top > 0] = -100
    for k in range(-100, 127):  # the least exponent that fits
        e = np.where((top > 0) & (top > 6 * 2.0 ** e) & (e == k), k + 1, e)
    y = np.where(finite[..., None], np.abs(np.where(np.isfinite(v), v, 0)) * 2.0 ** -e[..., None].astype(float), 0)
    hi = np.clip(np.searchsorted(GRID, y), 0, 7)
    lo = np.maximum(hi - 1, 0)
    below, above = y - GRID[lo], GRID[hi] - y
    q = np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)
    q = np.where(y == GRID[hi], hi, q) + np.where(np.signbit(v), 8, 0)
    q = np.where(finite[..., None], q, 0)
    return q.reshape(rows, nb * 32).astype(np.uint8), np.where(finite, e + 127, 255).astype(np.uint8)


def packed(q):
    return q[:, ::2] | q[:, 1::2] << 4


def codes(values):
    return np.stack([values & 15, values >> 4], -1).reshape(values.shape[0], -1)


def values(q, e, cols):
    v = GRID[q & 7] * np.where(q > 7, -1.0, 1.0)
    scale = np.where(e == 255, np.nan, 2.0 ** (e.astype(float) - 127))
    return (v * np.repeat(scale, 32, 1)[:, : v.shape[1]])[:, :cols]
