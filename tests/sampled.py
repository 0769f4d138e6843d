"""Sampling of a row by its definition in 64 bits."""
import numpy as np


def order_key(x):
    b = np.asarray(x, np.float32).view(np.int32).astype(np.int64)
    return np.where(b < 0, b ^ 0x7FFFFFFF, b)


def sample(logits, temperature, top_p, top_k, min_p, u):
    """(token, its share of the kept sum, how near the draw and the cuts are to the next token)."""
    l = np.asarray(logits, np.float32)
    ok = np.nonzero(np.isfinite(l))[0]
    if not temperature > 0 or not len(ok):
        x = np.where(np.isnan(l), -np.inf, l)
        return (int(np.argmax(x)) if (x > -np.inf).any() else 0), 1.0, 1.0
    f = np.float32
    order = ok[np.lexsort((ok, -order_key(l[ok])))]
    v = l[order].astype(np.float64)
    with np.errstate(all="ignore"):
        w = np.exp((v - v[0]) * (1 / float(f(temperature))))
    if 0 < top_k < len(w):
        w = w[:top_k]
    near = 1.0
    if f(top_p) < 1:
        s = np.cumsum(w)
        want = float(f(top_p)) * s[-1]
        n = int(np.searchsorted(s, want)) + 1
        near = min(near, np.abs(s - want).min() / s[-1])
        w = w[:max(1, n)]
    if f(min_p) > 0:
        n = int((w >= float(f(min_p))).sum())
        if not (w == float(f(min_p))).any():
            near = min(near, np.abs(w - float(f(min_p))).min())
        w = w[:max(1, n)]
    s = np.cumsum(w)
    u = float(f(u)) if u > 0 else 0.0
    want = min(u, 1 - 2.0 ** -24) * s[-1]
    if want > 0:
        near = min(near, np.abs(s - want).min() / s[-1])
    i = min(int(np.searchsorted(s, want, side="right")), len(w) - 1)
    return int(order[i]), w[i] / s[-1], near
