"""f64 oracle of the 8-bit projections and of the choice of tokens (test infrastructure only): plain
restatements of what include/tk_cuda.h says of tk_add_rmsnorm_fp8, tk_fp8_quantize, tk_fp8_matmul and
tk_sample_tokens.
"""
from __future__ import annotations

import numpy as np

BLOCK, LARGEST, LEAST = 128, 448.0, 2.0**-126


def decode_table():
    """The 256 values of e4m3: 1.mmm * 2^(e-7), 0.mmm * 2^-6 where e is 0, NaN where all seven bits are set."""
    code = np.arange(256)
    e, m = code >> 3 & 15, code & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m / 8 * 2.0**-6)
    v = np.where((code & 127) == 127, np.nan, v)
    return np.where(code & 128, -v, v)


TABLE = decode_table()


def add_rmsnorm(x, residual, weight, eps):
    """(sum, y) in f64."""
    s = np.asarray(x, np.float64) + (0 if residual is None else np.asarray(residual, np.float64))
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    return s, y if weight is None else y * np.asarray(weight, np.float64)


def group_scales(y, block_rows):
    """scales [ceil(rows / block_rows)][ceil(dim / 128)] in f64; NaN where a group is not finite."""
    rows, dim = y.shape
    out = np.zeros((-(-rows // block_rows), -(-dim // BLOCK)))
    for i in range(out.shape[0]):
        for j in range(out.shape[1]):
            g = y[i * block_rows:(i + 1) * block_rows, j * BLOCK:(j + 1) * BLOCK]
            out[i, j] = max(np.abs(g).max() / LARGEST, LEAST) if np.isfinite(g).all() else np.nan
    return out


def spread(scales, rows, dim, block_rows):
    """The scale of each value."""
    return np.repeat(np.repeat(scales, block_rows, 0)[:rows], BLOCK, 1)[:, :dim]


def matmul(a, a_scales, w, w_scales):
    """(out, size): the product of the values in f64, and that of their magnitudes, the scale of rounding errors."""
    av = TABLE[a] * spread(np.asarray(a_scales, np.float64), *a.shape, 1)
    wv = TABLE[w] * spread(np.asarray(w_scales, np.float64), *w.shape, BLOCK)
    return av @ wv.T, np.abs(av) @ np.abs(wv).T


def sample(logits, temperature, top_k, top_p, min_p, random):
    """(token, kept, slack) of one row; slack: how near (as a share of the sum) a comparison came to going the other way."""
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    if (l == -np.inf).all():
        return -1, 0, 1.0
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if l[order[0]] == np.inf:
        order = order[l[order] == np.inf]
    heat = 1.0 if temperature is None else float(temperature)
    if not heat > 0:
        return int(order[0]), 1, 1.0
    if top_k is not None and top_k > 0:
        order = order[:top_k]
    top = l[order[0]]
    t = np.where(l[order] == top, 0.0, (l[order] - top) / heat) if np.isfinite(top) else np.zeros(len(order))
    w = np.where(t * np.log2(np.e) < -999.8, 0.0, np.exp(t))
    count, slack = len(order), 1.0
    if top_p is not None and top_p < 1:
        goal, passed = max(float(top_p), 0.0) * w.sum(), np.cumsum(w)
        count = min(count, 1 + int(np.searchsorted(passed, goal)))
        if goal > 0:
            slack = min(slack, np.abs(passed - goal).min() / w.sum())
    if min_p is not None and min_p > 0:
        count = min(count, int((w >= min(float(min_p), 1.0)).sum()))
    by_index = np.argsort(order[:count])
    at, passed = order[by_index], np.cumsum(w[by_index])
    u = float(random)
    u = min(u, 1.0) if u > 0 else 0.0
    if 0 < u < 1:
        slack = min(slack, np.abs(passed - u * passed[-1]).min() / passed[-1])
    there = np.nonzero(w[by_index] > 0)[0]
    i = min(int(np.searchsorted(passed, u * passed[-1], side="right")), there[-1])
    return int(at[i]), count, slack
