"""Log probabilities, entropies, alternatives and gradients from their definition in 64 bits, with what float32 may lose of them."""
import numpy as np

U = 2.0**-24


def order(z, top):
    """Ids of a row's first `top` alternatives: NaN, then the largest, of equal ones the lowest index; -1 for none."""
    key = np.where(np.isnan(z), np.inf, z)
    ids = np.lexsort((np.arange(len(z)), -key, ~np.isnan(z)))[:top]
    return np.where(z[ids] == -np.inf, -1, ids).astype(np.int64)


def row(z, known, temperature, gl, gh, top):
    """(chosen, entropy, ids, log probabilities of them, gradient) of one row in 64 bits, and bounds of float32's errors for each
    but the ids.

    With d = (z - max) / T: a logit's exponent has three roundings (difference, factor, its product), so e_j is off by
    (3 |d_j| + 2) U relatively (the hardware's exponential to a unit in the last place); a thread adds up to 129 of them and a dozen
    more sums follow: 150 U. s so is off by S = (150 + 3 A) U with A = sum q |d|; ln s by that and 2 U of itself."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top_ids = order(z, top)
        odd = np.isnan(z).any() or (z == np.inf).any()
        shut = (z == -np.inf).all()
        if odd or shut:
            nan = np.nan if odd else -np.inf
            logs = np.where(top_ids >= 0, np.nan, -np.inf)
            grad = np.full(len(z), np.nan if odd else 0.0)
            if gl == 0 and gh == 0:
                grad[:] = 0
            none = np.zeros(len(z))
            return (nan if known >= 0 else 0.0, np.nan if odd else 0.0, top_ids, logs, grad), (0.0, 0.0, np.zeros(top), none)
        d = (z - z.max()) / temperature
        e = np.exp(d)
        s = e.sum()
        q = e / s
        size = np.where(q > 0, np.abs(d), 0.0)
        log_q = d - np.log(s)
        h = -(np.where(q > 0, q * log_q, 0.0)).sum()
        a, b = (q * size).sum(), (q * size * size).sum()
        off_s = (150 + 3 * a) * U + 2 * U * abs(np.log(s))
        off_log = np.where(z > -np.inf, 4 * U * np.abs(d) + off_s + U * np.abs(log_q), 0.0)
        # w's terms: e_j's own errors and two roundings, added up as s is; the quotient, its factor and the difference
        off_h = off_s + U * (156 * a + 3 * b + 4 * (a + np.log(s)))
        live_log = np.where(q > 0, log_q, 0.0)
        own = np.zeros(len(z))
        if known >= 0:
            own[known] = gl
        inner = np.where(q > 0, live_log + h, 0.0)
        grad = (own - gl * q - gh * q * inner) / temperature
        part = 160 * U + 3 * a * U + 4 * U * size  # e_j, 1 / s, the factors
        off_grad = q / temperature * (abs(gl) * part + abs(gh) * (np.abs(inner) * part + off_h + off_s + 6 * U * (h + np.log(s) + size)))
        off_grad = off_grad + 4 * U * np.abs(own) / temperature
        # e^d below float32's numbers is 0: what is lost of it
        off_grad = off_grad + 2.0**-126 * (abs(gl) + abs(gh) * 100) / temperature
        logs = np.where(top_ids >= 0, log_q[top_ids], -np.inf)
        off_top = np.where(top_ids >= 0, off_log[top_ids], 0.0)
        chosen = log_q[known] if known >= 0 else 0.0
        return (chosen, h, top_ids, logs, grad), (off_log[known] if known >= 0 else 0.0, off_h, off_top, off_grad)
