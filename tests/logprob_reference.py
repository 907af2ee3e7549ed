"""Plain 64-bit statements of the token log probabilities and their gradient,
with the error bounds the GPU tests compare against."""
from __future__ import annotations

import numpy as np

U32 = 2.0 ** -24            # unit roundoff of fp32
ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}   # half the spacing of subnormal results


def forward(x, tokens, temperature, top):
    """x [B, V] float64 (no NaN, no +inf). Per-row dict of arrays."""
    B, V = x.shape
    out = {k: np.zeros(B) for k in ("logprobs", "entropy", "max", "logsum", "ymax")}
    out["rank"] = np.full(B, -1, np.int64)
    out["top_ids"] = np.full((B, top), -1, np.int64)
    out["top_logprobs"] = np.full((B, top), -np.inf)
    ids = np.arange(V)
    for r in range(B):
        row, t = x[r], int(tokens[r])
        m = row.max()
        order = np.lexsort((ids, -row))[:top]
        out["max"][r] = m
        if t >= 0:
            out["rank"][r] = int((row > row[t]).sum() + (row[:t] == row[t]).sum())
        out["top_ids"][r, :len(order)] = order
        if m == -np.inf:                              # no distribution
            out["logsum"][r] = -np.inf
            out["logprobs"][r] = -np.inf if t >= 0 else 0.0
            continue
        y = (row - m) / temperature[r]
        e = np.exp(y)
        s = e.sum()
        lp = y - np.log(s)
        p = e / s
        keep = p > 0
        out["logsum"][r] = np.log(s)
        out["entropy"][r] = -(p[keep] * lp[keep]).sum()
        out["logprobs"][r] = lp[t] if t >= 0 else 0.0
        out["top_logprobs"][r, :len(order)] = lp[order]
        # the largest |y| whose term counts in fp32
        out["ymax"][r] = np.abs(y[e > 2.0 ** -40 * 1.0]).max()
    return out


def sum_bound(V, ymax):
    """Relative error of a row's sum of exp: every accumulator takes at most V / 128 + 64 terms one after
    another (a row has at least 128 accumulators, and a tree joins them), each term is exp of an argument
    with three roundings of relative size U32 plus an exp good to 4 U32, and the terms below 2^-40 that an
    implementation may drop or misjudge weigh at most V 2^-40 together."""
    return U32 * (V / 128 + 64 + 3 * ymax + 4) + V * 2.0 ** -40


def logprob_bound(V, ymax, lp):
    """|error| of a log probability: its own argument (at most eight roundings of its size, constants
    among them) plus the log sum's."""
    return 8 * U32 * np.abs(lp) + sum_bound(V, ymax) + 4 * U32 * np.log(V + 1.0)


def entropy_bound(V, ymax):
    """H = L - Q / S: Q's terms have one sign, so its relative error is that of a sum plus one product; the
    quotient is at most log V + ymax in size."""
    size = np.log(V + 1.0) + 1.0
    return (2 * sum_bound(V, ymax) + 8 * U32) * size + 4 * U32 * size


def gradient(x, tokens, temperature, grad_logprobs, grad_entropy):
    """d(sum(g lp) + sum(h H))/dx in 64 bits, and the magnitudes its terms have before they cancel."""
    B, V = x.shape
    d = np.zeros((B, V))
    size = np.zeros((B, V))
    for r in range(B):
        t = int(tokens[r])
        g = float(grad_logprobs[r]) if t >= 0 else 0.0
        h = float(grad_entropy[r]) if grad_entropy is not None else 0.0
        m = x[r].max()
        if (g == 0.0 and h == 0.0) or m == -np.inf:
            continue
        y = (x[r] - m) / temperature[r]
        lp = y - np.log(np.exp(y).sum())
        p = np.exp(lp)
        lp0 = np.where(p > 0, lp, 0.0)
        H = -(p * lp0).sum()
        d[r] = (-g * p - h * p * (lp0 + H)) / temperature[r]
        size[r] = p * (abs(g) + abs(h) * (np.abs(lp0) + H)) / temperature[r] * (np.abs(lp0) + 4)
        if t >= 0:
            d[r, t] += g / temperature[r]
            size[r, t] += 4 * abs(g) / temperature[r]
    return d, size


def gradient_bound(d, size, V, ymax, dtype):
    """One rounding to the result's type, plus fp32 arithmetic on terms of the given size: the argument of
    exp carries four roundings of its own size (counted in `size`) and the saved log sum one of log V's.
    Probabilities below 2^-126 may be flushed to zero: with the tests' factors (up to 2^8, times 2^7 for
    log p) that is 2^-111."""
    return (np.abs(d) * ROUND[dtype] + TINY[dtype]
            + U32 * size * (8 + np.log(V + 1.0)) + 2.0 ** -111)
