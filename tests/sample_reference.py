"""Plain 64-bit restatement of fp4_decode.sample, row by row on the host.  Nothing here calls the library."""
import numpy as np


def draw(logits, u, temperature, top_k, top_p, min_p):
    """(token, its share) of one row: logits as float64 numpy, settings as numbers (float32 values)."""
    l = np.where(np.isnan(logits), -np.inf, logits)
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if not len(order):
        return -1, 0.0
    if not temperature > 0:
        return int(order[0]), 1.0
    top = l[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(l[order] == top, 1.0, np.exp((l[order] - top) / temperature if np.isfinite(top) else np.full(len(order), -np.inf)))
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        sums = np.cumsum(w)
        w = w[: max(1, int(np.sum(np.concatenate(([0.0], sums[:-1])) < top_p * sums[-1])))]
    if min_p > 0:
        w = w[: max(1, int(np.sum(w >= min_p)))]
    sums = np.cumsum(w)
    u = min(float(u), 1.0 - 2.0 ** -24) if u > 0 else 0.0
    at = int(np.sum(sums <= u * sums[-1]))
    return int(order[at]), float(w[at] / sums[-1])
