"""Filtered draws written out plainly in 64 bits (numpy)."""
import numpy as np


def kept(x, temperature, top_k, top_p, min_p):
    """(weights float64 [V], 0 for what the filters take out) of one row of float32 logits."""
    x = np.asarray(x, dtype=np.float64)
    real = ~np.isnan(x)
    top = x[real].max()
    w = np.zeros(len(x))
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        z = (x - top) / float(np.float32(temperature))
        w[real] = np.where(x[real] == top, 1.0, np.exp(z[real]))
    order = np.nonzero(real)[0]
    order = order[np.lexsort((order, -x[order]))]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(w[order])
        order = order[(mass - w[order]) < float(np.float32(top_p)) * mass[-1]]
    order = order[w[order] >= float(np.float32(min_p))] if min_p > 0 else order
    out = np.zeros(len(x))
    out[order] = w[order]
    return out


def draw(x, temperature, top_k, top_p, min_p, u):
    """(id, distance of u from the nearest border between two ids as a part of the mass)."""
    if temperature == 0:
        return int(np.nanargmax(np.asarray(x, dtype=np.float64))), 1.0
    mass = np.cumsum(kept(x, temperature, top_k, top_p, min_p))
    at = u * mass[-1]
    i = int(np.searchsorted(mass, at, side="right"))
    i = min(i, len(mass) - 1)
    return i, float(np.abs(mass - at).min() / mass[-1])
