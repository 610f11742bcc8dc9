"""The label-selection operators in plain 64-bit numpy, row by row, from their definitions (test infrastructure)."""
import numpy as np


def rows_of(x):
    """[N, C, ...] -> [rows, C]"""
    return np.moveaxis(np.asarray(x), 1, -1).reshape(-1, x.shape[1])


def order_of(z):
    """Labels by score, larger first, the lower label first among equals, NaN before everything."""
    return np.lexsort((np.arange(z.size), np.where(np.isnan(z), -np.inf, -z), ~np.isnan(z)))


def logsumexp(b):
    b = np.asarray(b, np.float64)
    if b.size == 0:
        return -np.inf
    if np.isnan(b).any():
        return np.nan
    m = b.max()
    if not np.isfinite(m):
        return m
    return m + np.log(np.exp(b - m).sum())


def top(z, k, t):
    o = order_of(z)
    return z[o[:k]], o[:k], logsumexp(z[o[k:]] / t)


def distill(z, values, labels, rest, t, valid=True):
    """(loss, gradient, bound): bound = what an error of one unit in every exponent can do to (loss, gradient)."""
    C = z.size
    zero = (0.0, np.zeros(C), (0.0, np.zeros(C)))
    use = [(float(v) / t, int(c)) for v, c in zip(values, labels) if 0 <= c < C]
    a = np.array([v for v, _ in use] + ([] if rest is None else [float(rest)]), np.float64)
    if not valid or not use or logsumexp(a) == -np.inf or (z == -np.inf).all():
        return zero
    named = sorted({c for _, c in use})
    with np.errstate(invalid="ignore", divide="ignore"):
        b = z.astype(np.float64) / t
        b = b - (b.max() if np.isfinite(b.max()) else 0.0)     # (next to a score of -3e38 a logarithm is lost in 64 bits too)
        Z = logsumexp(b)
        logq = b - Z
        outside = np.ones(C, bool)
        outside[named] = False
        tail = logsumexp(b[outside]) - Z
        logp = a - logsumexp(a)
        student = np.array([logq[c] for _, c in use] + ([] if rest is None else [tail]))
        p = np.exp(logp)
        terms = np.where(p == 0, 0.0, p * (logp - student))
        size = np.where(p == 0, 0.0, p * (1 + np.abs(logp) + np.abs(student)))
        q = np.exp(logq)
        grad, scale = q.copy(), q.copy()
        for (_, c), pj in zip(use, p):
            grad[c] -= pj
            scale[c] += pj
        if rest is not None and outside.any() and tail != -np.inf:
            share = p[-1] * np.exp(logq[outside] - tail)
            grad[outside] -= share
            scale[outside] += share
        reach = 1 + np.where(np.isfinite(logq), np.abs(logq), 0.0)
    return t * t * terms.sum(), t * grad, (t * t * size.sum(), t * scale * reach)


def sample(z, u, t=1.0, top_k=0, top_p=1.0, min_p=0.0):
    C = z.size
    z = z.astype(np.float64)
    m = z.max()
    if not np.isfinite(m):
        return -1, -np.inf
    k = 1 if not t > 0 else (C if top_k <= 0 else min(top_k, C))
    with np.errstate(over="ignore"):
        w = np.exp((z - m) * (1.0 / t if t > 0 else 1.0))
    o = order_of(z)[:k]
    front = np.concatenate([[0.0], np.cumsum(w[o])])
    total = front[-1]
    keep = [c for i, c in enumerate(o) if i == 0 or ((front[i] < top_p * total or top_p >= 1) and w[c] >= min_p and w[c] > 0)]
    keep = sorted(keep)
    run = np.cumsum(w[keep])
    hit = np.nonzero(run > max(u, 0.0) * run[-1])[0]
    i = hit[0] if hit.size else len(keep) - 1
    return keep[i], float(np.log(w[keep[i]] / run[-1]))
