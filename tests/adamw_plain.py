"""AdamW and 8-bit moments from their definitions: a step in 64 bits with the bounds of its float32 roundings, and the held
moments bit by bit in float32 numpy, whose every operation rounds once."""
import numpy as np

HELD = 128
F = np.float32


def grid():
    """The 127 finite E4M3 magnitudes by code."""
    b = np.arange(127)
    field, low = b >> 3, b & 7
    return np.where(field == 0, low * 2.0**-9, (1 + low / 8) * 2.0 ** (field - 7.0))


def _blocks(x):
    return np.pad(x, (0, -len(x) % HELD)).reshape(-1, HELD)


def hold_first(m):
    """(codes, scales) of float32 moments."""
    with np.errstate(all="ignore"):
        m = _blocks(m.astype(F))
        finite = np.isfinite(m)
        top = np.where(finite, np.abs(m), F(0)).max(1)
        scale = np.maximum(top * F(1 / 448), F(2.0**-126))
        x = (m * (F(1) / scale)[:, None]).astype(np.float64)
    g = grid()
    y = np.minimum(np.abs(np.where(finite, x, 0)), 448)
    hi = np.clip(np.searchsorted(g, y), 0, 126)
    lo = np.maximum(hi - 1, 0)
    below, above = y - g[lo], g[hi] - y
    q = np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)
    q = np.where(y == g[hi], hi, q)
    q = np.where(finite, q, 127) + np.where(np.signbit(m), 128, 0)
    return q.astype(np.uint8).reshape(-1), scale


def first_values(codes, scale):
    g = np.append(grid(), np.nan)
    v = (g[codes & 127] * np.where(codes > 127, -1.0, 1.0)).astype(F).reshape(-1, HELD)
    return (v * scale[:, None]).reshape(-1)


def ratios():
    """What codes 0 to 254 of second moments stand for."""
    c = np.arange(255)
    at = c + 2
    return np.where(c == 0, 0.0, 2.0 ** (at // 8 - 32.0) * (1 + at % 8 / 8))


def hold_second(v):
    with np.errstate(all="ignore"):
        v = _blocks(v.astype(F))
        finite = np.isfinite(v)
        scale = np.maximum(np.where(finite, v, F(0)).max(1), F(2.0**-126))
        y = (v * (F(1) / scale)[:, None]).astype(np.float64)
    r = ratios()
    y = np.where(finite, y, 1.0)
    hi = np.clip(np.searchsorted(r, y), 1, 254)
    lo = np.maximum(hi - 1, 1)
    below, above = y - r[lo], r[hi] - y
    # the last of the three bits is 0 where (code + 2) is even
    q = np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)
    q = np.where(v > 0, q, 0)
    q = np.where(finite, q, 255)
    return q.astype(np.uint8).reshape(-1), scale


def second_values(codes, scale):
    r = np.append(ratios(), np.inf).astype(F)
    return (r[codes].reshape(-1, HELD) * scale[:, None]).reshape(-1)


def moments32(m, v, g, scale, rates):
    """The step's new moments in float32, operation by operation."""
    b1, b2 = rates["beta1"], rates["beta2"]
    with np.errstate(all="ignore"):
        x = g.astype(F) * F(scale)
        return F(b1) * m + F(1 - b1) * x, F(b2) * v + F(1 - b2) * (x * x)


def step(p, g, m, v, scale, t, rates):
    """(p, m, v) after a step in 64 bits and how far float32 roundings may take each of them."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    b1, b2, lr = rates["beta1"], rates["beta2"], rates["learning_rate"]
    x, u = g * scale, 2.0**-24
    m1, v1 = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
    # the scale, the factor's own rounding (half of a step at most, as every rounding), the product, the sum
    off_m = 4 * u * (np.abs(b1 * m) + np.abs((1 - b1) * x))
    off_v = 6 * u * v1  # the square has the scale's rounding twice
    rate, root = lr / (1 - b1**t), 1 / np.sqrt(1 - b2**t)
    den = np.sqrt(v1) * root + rates["epsilon"]
    change = rate * m1 / den
    decay = lr * rates["weight_decay"] * p
    # the denominator: half of v's 6, the root, its factor and product, epsilon and the sum: 8; the quotient; the rate's factor
    # and product: 2; the subtractions: half a step of what they leave, each
    off_p = rate * off_m / den + 12 * u * np.abs(change) + 3 * u * np.abs(decay) + 2 * u * (np.abs(p) + np.abs(change))
    return (p - decay - change, m1, v1), (off_p, off_m, off_v)
