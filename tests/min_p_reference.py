"""The min-p sampler's definition, row by row on the host in 64 bits (numpy).

Penalties and the division by the temperature are operations on 32-bit numbers
by the definition; everything after them is in 64 bits. `near` marks rows whose
draw or top-p cut lies within 1e-9 of the mass from a border between two
tokens, where 64-bit sums and sums of integers may part."""
from __future__ import annotations

from typing import NamedTuple

import numpy as np

F = np.float32


class Row(NamedTuple):
    id: int
    logprob: float
    kept: int
    near: bool
    kept_ids: np.ndarray
    probs: np.ndarray


def sample_row(x, u, min_p, temperature=1.0, top_k=0, top_p=1.0, greedy=False, rep=1.0, pres=0.0, freq=0.0,
               history=()) -> Row:
    """x: float32 values of the row's logits."""
    x = np.array(x, dtype=F)
    v = len(x)
    ids, counts = np.unique(np.asarray(history, dtype=np.int64), return_counts=True)
    if len(ids):
        old = x[ids]
        if F(rep) != 1:
            old = np.where(old > 0, old / F(rep), old * F(rep))
        if F(freq) != 0:
            old = old - F(freq) * counts.astype(F)
        if F(pres) != 0:
            old = old - F(pres)
        x[ids] = old
    if greedy or temperature == 0:
        at = int(np.argmax(x))       # the first maximum; NaN counts as one
        return Row(at, 0.0, 1, False, np.array([at]), np.ones(1))
    y = x / F(temperature) + F(0)
    order = np.lexsort((np.arange(v), -y.astype(np.float64)))
    ys = y[order].astype(np.float64)
    top = ys[0]
    keep = ys > -np.inf
    if min_p > 0:
        keep &= ys >= top + np.log(np.float64(F(min_p)))
    if 0 < top_k < v:
        keep &= ys >= ys[top_k - 1]
    n = int(keep.sum())
    mass = np.exp(ys[:n] - top)
    upto = np.cumsum(mass)
    near = False
    if top_p < 1:
        limit = np.float64(F(top_p)) * upto[-1]
        before = upto - mass
        near = bool((np.abs(before[1:] - limit) <= 1e-9 * upto[-1]).any())
        n = int((before <= limit).sum())
        mass, upto = mass[:n], upto[:n]
    target = np.float64(F(u)) * upto[-1]
    near = near or bool((np.abs(upto[:-1] - target) <= 1e-9 * upto[-1]).any())
    at = min(int(np.searchsorted(upto, target, side="right")), n - 1)
    return Row(int(order[at]), float(ys[at] - top - np.log(upto[-1])), n, near, order[:n], mass / upto[-1])
