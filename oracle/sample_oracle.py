"""The next token of a row of logits from its definition, in float64."""
import numpy as np


def kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens, weights): what is kept, by falling logit and rising number."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    order = order[np.isfinite(x[order]) | (x[order] > 0)]
    if not order.size:
        return order, np.zeros(0)
    if not temperature > 0:
        return order[:1], np.ones(1)
    if top_k > 0:
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    w = np.where(np.isnan(w), 0.0, w)
    if top_p < 1:
        n = max(1, int(np.count_nonzero(np.cumsum(w) - w < top_p * w.sum())))
        order, w = order[:n], w[:n]
    n = max(1, int(np.count_nonzero(w >= min(min_p, 1.0))))
    return order[:n], w[:n]


def sample(x, u, **settings):
    """(token, distance): distance is how far u is, as a share of the kept weight, from the next
    border between two tokens."""
    order, w = kept(x, **settings)
    if not order.size:
        return -1, 1.0
    by = np.argsort(order)
    mass = np.cumsum(w[by])
    share = mass / mass[-1]
    at = min(int(np.count_nonzero(share <= u)), len(share) - 1)
    edges = share[:-1]
    return int(order[by][at]), float(np.abs(edges - u).min()) if edges.size else 1.0
