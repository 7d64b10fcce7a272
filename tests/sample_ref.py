"""A draw of a token from its definition, row by row, in extended precision on the CPU
(tests/test_gpu_sample.py)."""
import math

import numpy as np


def draw(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, scale=1.0):
    """(token, probability it was drawn with, the least distance of u and of top_p's cut from
    a border between two tokens) of one row; every argument as a Python or numpy number."""
    l = np.asarray(logits, np.float64) * scale
    with np.errstate(invalid="ignore"):
        live = np.flatnonzero(l > -np.inf)        # (a NaN compares false)
    if live.size == 0:
        return -1, 0.0, 1.0
    order = live[np.lexsort((live, -l[live]))]
    if not temperature > 0:
        return int(order[0]), 1.0, 1.0
    top = l[order[0]]
    with np.errstate(invalid="ignore"):
        e = np.where(l[order] == top, 1.0, np.exp(((l[order] - top) / np.float64(temperature)).astype(np.longdouble)))
    if math.isinf(top):
        e = (l[order] == top).astype(np.longdouble)
    if 0 < top_k < l.size:
        order, e = order[:top_k], e[:top_k]
    border = 1.0
    if top_p < 1:
        mass = np.cumsum(e)
        cut = np.longdouble(top_p) * mass[-1]
        n = max(1, int(np.searchsorted(mass, cut, side="left")) + 1)
        border = float(np.abs(mass - cut).min() / mass[-1])
        order, e = order[:n], e[:n]
    if min_p > 0:
        keep = (e >= min_p) | (np.arange(e.size) == 0)
        order, e = order[keep], e[keep]
    at = np.argsort(order)
    order, e = order[at], e[at]
    mass = np.cumsum(e)
    u = 0.0 if not u > 0 else float(u)
    target = np.longdouble(u) * mass[-1]
    i = min(int(np.searchsorted(mass, target, side="right")), int(np.flatnonzero(e > 0)[-1]))
    return int(order[i]), float(e[i] / mass[-1]), min(border, float(np.abs(mass[:-1] - target).min() / mass[-1]) if i or mass.size > 1 else 1.0)
