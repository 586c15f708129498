"""The sampler's definition in 64 bits (numpy), and whether a token is decided
by less than the kernel's weights can tell apart."""
import numpy as np


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Token of one row, and the distance of the draw from the nearest border
    (relative to the whole mass)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, np.inf
    if not temperature > 0:
        return int(np.argmax(x)), np.inf
    fall = np.argsort(-x, kind="stable")
    fall = fall[x[fall] > -np.inf]
    if 0 < top_k < fall.size:
        fall = fall[:top_k]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[fall] == x.max(), 1.0, np.exp((x[fall] - x.max()) / np.float64(temperature)))
    near = np.inf
    if top_p < 1:
        run, goal = np.cumsum(w), max(top_p, 0.0) * w.sum()
        n = 1 + int(np.searchsorted(run, goal, "left"))
        near = min(near, float(np.abs(run - goal).min() / w.sum()))
        fall, w = fall[:n], w[:n]
    if min_p > 0:
        ok = w >= min(min_p, 1.0)
        fall, w = fall[ok], w[ok]
    order = np.argsort(fall)
    fall, run = fall[order], np.cumsum(w[order])
    goal = min(max(u, 0.0), 1.0) * run[-1]
    i = min(int(np.searchsorted(run, goal, "right")), int(np.flatnonzero(w[order] > 0)[-1]))
    near = min(near, float(np.abs(run - goal).min() / run[-1])) if u > 0 else near
    return int(fall[i]), near
