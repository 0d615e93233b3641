"""Tokens drawn from logits by given random numbers, in float64 from the definition (test infrastructure; csrc/sample.hip is checked against it)."""

from __future__ import annotations

import numpy as np


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """one row -> token, its probability, how near (relative to the whole) the borders that were decided lie to another outcome.  x: float64 values of the logits; the settings as 32 bits hold them"""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    if not (temperature >= 0 and top_p >= 0 and min_p >= 0) or not (x > -np.inf).any():
        return -1, 0.0, 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if temperature == 0:
        return int(order[0]), 1.0, 1.0
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        z = np.where(x == top, 0.0, (x - top) / temperature if top < np.inf else -np.inf)
    w = np.exp(z)
    near = 1.0
    if 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(w[order])
        n = int(np.searchsorted(mass, top_p * mass[-1], side="left")) + 1
        near = min(near, np.abs(mass - top_p * mass[-1]).min() / mass[-1])
        order = order[: max(1, min(n, len(order)))]
    keep = np.zeros(len(x), bool)
    keep[order] = True
    with np.errstate(divide="ignore"):
        least = np.log(np.float64(min_p))
    if min_p > 0:
        near = min(near, np.abs(z[order] - least).min() if min_p != 1 else 1.0)
    keep &= (z >= least) | (z == 0)
    mass = np.cumsum(np.where(keep, w, 0.0))
    at = min(max(u if u == u else 0.0, 0.0), 1.0) * mass[-1]
    hits = np.flatnonzero(keep & (mass > at))
    token = int(hits[0]) if len(hits) else int(np.flatnonzero(keep & (w > 0))[-1])
    if 0 < u < 1:
        near = min(near, np.abs(mass - at).min() / mass[-1])
    return token, w[token] / mass[-1], near
