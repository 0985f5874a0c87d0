"""The sampler's definition in 64 bits (test infrastructure): one row at a time, by a sort."""
import numpy as np


NEAR = 1e-9


def row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """(index, probability, margin): margin is how far u or min_p is from where the answer changes,
    relative to the row's mass, and 0 where moving the limit of top_p by NEAR of the mass changes it;
    below NEAR two right evaluations may differ."""
    i, p, margin = _row(x, u, temperature, top_k, top_p, min_p, mask, 0.0)
    if top_p < 1:
        for shift in (-NEAR, NEAR):
            if _row(x, u, temperature, top_k, top_p, min_p, mask, shift)[0] != i:
                margin = 0.0
    return i, p, margin


def _row(x, u, temperature, top_k, top_p, min_p, mask, shift):
    x = np.asarray(x, np.float64).copy()
    n = x.size
    if mask is not None:
        x[np.asarray(mask) != 0] = -np.inf
    if np.isnan(x).any():
        return -1, np.nan, 1.0
    live = np.nonzero(x > -np.inf)[0]
    if not live.size:
        return -1, 0.0, 1.0
    t, p, q = (float(np.float32(v)) for v in (temperature, top_p, min_p))
    u = float(np.float32(u))
    u = min(u, float(np.float32(0.99999994))) if u > 0 else 0.0
    p = 1.0 if not p < 1 else max(p, 0.0)
    q = 0.0 if not q > 0 else min(q, 1.0)
    order = live[np.lexsort((live, -x[live]))]
    top = x[order[0]]
    if not t > 0:
        return int(order[0]), 1.0, 1.0
    if top == np.inf:
        w = (x[order] == np.inf).astype(np.float64)
    else:
        with np.errstate(over="ignore"):
            w = np.exp((x[order] - top) / t)
    margin = 1.0
    if 0 < top_k < order.size:
        order, w = order[:top_k], w[:top_k]
    keep = np.ones(order.size, bool)
    if p < 1:
        s1 = w.sum()
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep = before < (p + shift) * s1
        keep[0] = True
    if q > 0:
        keep &= w >= q
        far = np.abs(w - q)
        margin = min(margin, far[w < 1].min() if (w < 1).any() else 1.0)
    order, w = order[keep], w[keep]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    upto = np.cumsum(w)
    s = upto[-1]
    at = min(int(np.searchsorted(upto, u * s, side="right")), order.size - 1)
    while w[at] == 0:
        at -= 1
    if u > 0:
        margin = min(margin, np.abs(upto - u * s).min() / s)
    return int(order[at]), float(w[at] / s), margin
