"""Plain 64-bit forms of the training operators, with bounds of their f32
kernels' errors (U = 2^-24, a rounding's share in f32)."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24
EPS = 1e-5
BLOCK = 32
E4M3 = np.array([np.ldexp(m, -9) if e == 0 else np.ldexp(8 + m, e - 10)
                 for e in range(16) for m in range(8) if not (e == 15 and m == 7)])  # 0 .. 448, ascending


# --- embedding -----------------------------------------------------------------
def centered(x):
    """(c, r, slack): rows less their mean, 1 / sqrt(var + eps), and how far
    the kernel's centered row may lie from c.

    A row's sum adds at most 4 neighbours, 8 such and 6 exchanges of a wave: 16
    roundings of its values' magnitudes, 17 with the division.  The first mean is
    off by 17 U mean|x|, a shift that the second one takes out but for its
    own 17 U of what is left; each difference rounds."""
    c = x - x.mean(1, keepdims=True)
    r = 1 / np.sqrt((c * c).mean(1, keepdims=True) + EPS)
    shift = 17 * U * np.abs(x).mean(1, keepdims=True)
    slack = 2 * U * (np.abs(c) + shift) + 18 * U * (np.abs(c).mean(1, keepdims=True) + shift)
    return c, r, slack


def embed(tokens, table, scale, norm, eps):
    """(rows, bound)."""
    V, D = table.shape
    there = (tokens >= 0) & (tokens < V)
    out, bound = np.zeros((tokens.size, D)), np.zeros((tokens.size, D))
    x = table[tokens[there]]
    if norm:
        c, r, slack = centered(x)
        out[there] = scale * c * r
        # r: half the variance's error (a sum of squares, 2 * 20 U of it) and a few roundings.
        bound[there] = np.abs(out[there]) * 44 * U + abs(scale) * r * slack
    else:
        out[there] = scale * x
        bound[there] = np.abs(out[there]) * U
    return out, bound + np.abs(out) * eps / 2 + 1e-40


def embed_vjp(grad, tokens, table, scale, norm, eps, old=None):
    V, D = table.shape
    there = (tokens >= 0) & (tokens < V)
    s, mag, n = np.zeros((V, D)), np.zeros((V, D)), np.zeros((V, 1))
    np.add.at(s, tokens[there], grad[there])
    np.add.at(mag, tokens[there], np.abs(grad[there]))
    np.add.at(n, tokens[there], 1.0)
    s *= scale
    # A sum of n rows rounds n times, a few more where runs are joined and scaled.
    off = (n + 8) * U * mag * abs(scale)
    if norm:
        c, r, slack = centered(table)
        xh = c * r
        X = 44 * U * np.abs(xh) + r * slack
        mean = lambda v: v.mean(1, keepdims=True)  # noqa: E731
        size = np.abs(s) + mean(np.abs(s)) + np.abs(xh) * mean(np.abs(s * xh))
        off = r * (off + mean(off) + np.abs(xh) * mean(off * np.abs(xh)) + X * mean(np.abs(s * xh))
                   + np.abs(xh) * mean(np.abs(s) * X) + 64 * U * size)
        s = r * (s - mean(s) - xh * mean(s * xh))
        s[n[:, 0] == 0] = 0.0
        off[n[:, 0] == 0] = 0.0
    if old is not None:
        s = s + old
        off = off + U * np.abs(s)
    return s, off + np.abs(s) * eps / 2 * ((n > 0) | (old is None)) + 1e-40


# --- 8 bits -------------------------------------------------------------------------
def powers(x):
    """e of each block of 32 of the rows x [rows, C] (finite magnitudes)."""
    rows, C = x.shape
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    a = np.pad(a, ((0, 0), (0, -C % BLOCK))).reshape(rows, -1, BLOCK).max(2)
    m, k = np.frexp(a)                       # a = m 2^k, m in [1/2, 1); 448 = 0.875 2^9
    return np.maximum(np.where(a > 0, np.where(m > 0.875, k + 1, k) - 9, -117), -117)


def in8(x):
    """(values, e): x [rows, C] as its nearest e4m3 of each block, ties to even;
    past 240 * 2^120, where the next codes are no finite f32, as that."""
    e = powers(x)
    x = np.where(np.isfinite(x), np.clip(x, -240 * 2.0 ** 120, 240 * 2.0 ** 120), x)
    p = np.ldexp(1.0, np.repeat(e, BLOCK, 1)[:, :x.shape[1]])
    w = np.abs(x) / p
    at = np.clip(np.searchsorted(E4M3, np.where(np.isfinite(w), w, 0.0)), 1, len(E4M3) - 1)
    low, high = E4M3[at - 1], E4M3[at]
    middle = (low + high) / 2
    up = (w > middle) | ((w == middle) & (at % 2 == 0))   # (an even code is an even index)
    v = np.copysign(np.where(up, high, low) * p, x)
    return np.where(np.isfinite(x), v, np.nan), e


# --- gated block ------------------------------------------------------------------------
def _erf(x):
    from scipy.special import erf
    return erf(x)


def act(kind, q):
    """(act(q), act'(q))."""
    if kind == "relu":
        return np.where(q > 0, q, 0.0), (q > 0).astype(float)
    if kind == "silu":
        z = 1 / (1 + np.exp(-q))
        return q * z, z * (1 + q * (1 - z))
    z = 0.5 * (1 + _erf(q / np.sqrt(2)))
    return q * z, z + q * np.exp(-q * q / 2) / np.sqrt(2 * np.pi)


def up(kind, p):
    return act("relu", p) if kind == "relu" else (p, np.ones_like(p))


def project(x, c, wu, wg, th):
    """(p, q, dp, dq) [H, M, N], the last two how far f32 sums may be off: a sum of D
    products rounds D times, the difference with th once."""
    H, D, N = wu.shape
    p = np.stack([x @ wu[h] for h in range(H)])
    q = np.stack([c[h] @ wg[h] for h in range(H)])
    mp = np.stack([np.abs(x) @ np.abs(wu[h]) for h in range(H)])
    mq = np.stack([np.abs(c[h]) @ np.abs(wg[h]) for h in range(H)])
    return p - th, q - th, (D + 2) * U * (mp + abs(th)), (D + 2) * U * (mq + abs(th))


# An activation's and its slope's own errors: exp, erf, reciprocal and the products, a
# dozen roundings of values up to their magnitudes (|q|, 1 + |q|).
ACT_OFF = 16 * U


def forward(kind, p, q, op, oq, m):
    """(out, bound) from projections and their errors; slopes are at most 1.13."""
    u, _ = up(kind, p)
    a, _ = act(kind, q)
    out = u * a * m * m
    own = 0.0 if kind == "relu" else ACT_OFF * np.abs(q)
    off = m * m * (op * (np.abs(a) + 1.13 * oq) + np.abs(u) * (1.13 * oq + own)) + 8 * U * np.abs(out)
    return out, off


def backward(kind, g, x, c, wu, wg, p, q, op, oq, m):
    """{name: (value, bound)} for g [H, M, N], from projections and their errors (0: as
    given).  dp and dq round to bf16 (2^-8 of them) before the products."""
    H = p.shape[0]
    u, du = up(kind, p)
    a, da = act(kind, q)
    gm = np.abs(g) * m * m
    dp, dq = g * m * m * a * du, g * m * m * u * da
    own = 0.0 if kind == "relu" else ACT_OFF * (1 + np.abs(q))
    # The slope's own slope is at most 1.13; relu's jumps where the sign is not certain.
    odp = gm * np.abs(du) * (1.13 * oq + own * np.abs(q))
    odq = gm * (op * np.abs(da) + (np.abs(u) + op) * (0.0 if kind == "relu" else 1.13 * oq + own))
    if kind == "relu":
        odp += np.where((np.abs(p) <= op) & (op > 0), gm * (np.abs(a) + oq), 0.0)
        odq += np.where((np.abs(q) <= oq) & (oq > 0), gm * (np.abs(u) + op), 0.0)
    odp += (2.0 ** -8 + 8 * U) * np.abs(dp) + 2.0 ** -8 * odp + 1e-38
    odq += (2.0 ** -8 + 8 * U) * np.abs(dq) + 2.0 ** -8 * odq + 1e-38
    N, M = p.shape[2], p.shape[1]

    def product(l, r, lo=None, ro=None, terms=0):
        """l @ r, where l or r is off by lo or ro, in f32 sums of `terms` products."""
        lo = np.zeros_like(l) if lo is None else lo
        ro = np.zeros_like(r) if ro is None else ro
        mag = (np.abs(l) + lo) @ (np.abs(r) + ro)
        return l @ r, lo @ (np.abs(r) + ro) + np.abs(l) @ ro + (terms + 8) * U * mag
    out = {"up": [], "gate": [], "context": []}
    dx = dxo = 0.0
    for h in range(H):
        v, o = product(dp[h], wu[h].T, lo=odp[h], terms=N + 64)
        dx, dxo = dx + v, dxo + o + U * H * np.abs(v)
        out["context"].append(product(dq[h], wg[h].T, lo=odq[h], terms=N + 64))
        out["up"].append(product(x.T, dp[h], ro=odp[h], terms=M + 64))
        out["gate"].append(product(c[h].T, dq[h], ro=odq[h], terms=M + 64))
    out = {k: tuple(np.stack(t) for t in zip(*v)) for k, v in out.items()}
    out["current"] = (dx, dxo)
    return out
