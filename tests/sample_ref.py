"""Sampling of rows in float64 numpy, written from its definition."""
import numpy as np


def sample(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """(token, share) of one row."""
    x = np.asarray(x).astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    best = int(x.argmax())
    if x[best] == -np.inf:
        return -1, 0.0
    if not np.float32(temperature) >= np.float32(1e-6):
        return best, 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x[best], 1.0, np.exp(np.where(np.isneginf(x), -np.inf, (x - x[best]) / np.float64(np.float32(temperature)))))
    order = np.lexsort((np.arange(x.size), -x))
    order = order[w[order] >= min(1.0, float(np.float32(min_p)))]
    if top_k > 0:
        order = order[:top_k]
    p = float(np.float32(top_p))
    if p < 1:
        mass = np.cumsum(w[order])
        order = order[np.concatenate([[True], mass[:-1] < p * mass[-1]])]
    left = np.sort(order)
    run = np.cumsum(w[left])
    t = int(left[np.nonzero(run > float(np.float32(u)) * run[-1])[0][0]])
    return t, w[t] / run[-1]
