"""Sampling in 64 bits, one row at a time, from the definition: the oracle of
the sample_tokens tests."""
import math

import numpy as np

LEAST = -42.0 * math.log(2.0)
F32_MAX = float(np.finfo(np.float32).max)


def kept_weights(x, temperature, top_k, top_p, min_p):
    """(indices in order, their weights after all cuts) of one row, or None.
    The settings are f32 values, as the library takes them."""
    temperature, top_p, min_p = (np.float64(np.float32(v)) for v in (temperature, top_p, min_p))
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    x[x == np.inf] = F32_MAX
    real = np.flatnonzero(x > -np.inf)
    if real.size == 0:
        return None
    order = real[np.lexsort((real, -x[real]))]
    if not temperature > 0:
        return order[:1], np.ones(1)
    if 0 < top_k < order.size:
        order = order[:top_k]
    with np.errstate(over="ignore"):
        d = (x[order] - x[order[0]]) / temperature
    w = np.where(d < LEAST, 0.0, np.exp(d))
    kept = np.ones(order.size, bool)
    if top_p < 1:
        kept = np.concatenate([[0.0], np.cumsum(w)[:-1]]) < top_p * w.sum()
        kept[0] = True
    if min_p > 0:
        kept &= w >= min(min_p, 1.0)
    return order, np.where(kept, w, 0.0)


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    got = kept_weights(x, temperature, top_k, top_p, min_p)
    if got is None:
        return -1, -math.inf
    order, w = got
    by_index = np.argsort(order)
    sums = np.cumsum(w[by_index])
    u = min(max(float(u), 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    at = by_index[min(int(np.searchsorted(sums, u * sums[-1], side="right")), order.size - 1)]
    return int(order[at]), math.log(w[at] / w.sum())


def sample(x, u, **kw):
    """Row by row; settings are numbers or one a row."""
    rows = len(u)
    pick = {k: (np.asarray(v) if np.ndim(v) else np.full(rows, v)) for k, v in kw.items()}
    got = [sample_row(x[r], u[r], **{k: v[r] for k, v in pick.items()}) for r in range(rows)]
    return np.array([g[0] for g in got], np.int32), np.array([g[1] for g in got])
