"""Plain 64-bit forms of the paged-cache operators and of the sampling operator, one row at a time (numpy)."""
import numpy as np


def rotate_normed(x, w, pos, base, eps):
    """x [heads, head_dim] at one position: RMS norm with w (None: none), then the rotation of the pairs (i, i + half)."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    half = x.shape[-1] // 2
    a = pos * float(base) ** (-np.arange(half, dtype=np.float64) / half)
    c, s = np.cos(a), np.sin(a)
    return np.concatenate([x[..., :half] * c - x[..., half:] * s, x[..., :half] * s + x[..., half:] * c], -1)


def seen(pos, window, n_sink):
    """Positions that position ``pos`` attends to."""
    j = np.arange(pos + 1)
    return j[(j > pos - window) | (j < n_sink)] if window else j


def attend(q, k, v, pos, window, n_sink, scale, cap):
    """q [heads, d] at position pos, k and v [positions, kv_heads, d]: outputs [heads, d], and the largest |score| before the cap."""
    j, group = seen(pos, window, n_sink), q.shape[0] // k.shape[1]
    out, most = np.empty(q.shape, np.float64), 0.0
    for h in range(q.shape[0]):
        s = k[j, h // group].astype(np.float64) @ q[h].astype(np.float64) * scale
        most = max(most, float(np.abs(s).max()))
        if cap:
            s = cap * np.tanh(s / cap)
        p = np.exp(s - s.max())
        out[h] = p @ v[j, h // group].astype(np.float64) / p.sum()
    return out, most


def sample(logits, temperature, top_k, top_p, min_p, u):
    """The token, or -1, in extended precision; second: its distance from another outcome of the draw or of the nucleus,
    relative to the sums that decide (1 where all weights are 0 or 1: sums of those have no rounding)."""
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.longdouble)
    alive = np.flatnonzero(x > -np.inf)
    if not len(alive):
        return -1, 1.0
    best = x.max()
    order = alive[np.argsort(-x[alive], kind="stable")]
    if not temperature > 0:
        return int(order[0]), 1.0
    w = np.zeros(len(x), np.longdouble)
    w[alive] = 1.0 if np.isinf(temperature) and np.isfinite(best) else np.where(x[alive] == best, 1.0, np.exp((x[alive] - best if np.isfinite(best) else -np.inf) / np.longdouble(temperature)))
    margin = 1.0
    if top_k:
        order = order[:top_k]
    if top_p < 1:
        c = np.cumsum(w[order])
        t = max(np.longdouble(top_p), 0) * c[-1]
        n = int(np.searchsorted(c, t, side="left")) + 1
        margin = min(margin, float(np.abs(c - t).min() / c[-1])) if top_p > 0 else margin
        order = order[:n]
    order = np.sort(order[w[order] >= min(min_p, 1.0)])
    c = np.cumsum(w[order])
    t = np.longdouble(u) * c[-1]
    margin = min(margin, float(np.abs(c - t).min() / c[-1]))
    if np.isin(w, (0, 1)).all():
        margin = 1.0
    return int(order[min(int(np.searchsorted(c, t, side="right")), len(order) - 1)]), margin
