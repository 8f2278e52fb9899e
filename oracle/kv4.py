"""f64 oracle of the serving-step operators over the 4-bit key/value cache (test infrastructure only).

Plain restatements, loop by loop, of what include/tk_cuda.h says of tk_paged_slots, tk_qk_norm_rope,
tk_kv4_append / tk_kv4_gather and tk_kv4_attention.
"""
from __future__ import annotations

import numpy as np


def paged_slots(ctx, new, free_blocks, free_range, tables, block_size, num_blocks, max_tokens):
    """(tables, kv_lens, query_start, positions, slots, counts) after the step."""
    tables = np.array(tables, dtype=np.int32)
    batch, max_blocks = tables.shape
    begin, end = max(int(free_range[0]), 0), int(free_range[1])
    kv, start = np.zeros(batch, np.int32), np.zeros(batch + 1, np.int32)
    pos = np.full(max_tokens, -1, np.int32)
    slots = np.full(max_tokens, -1, np.int32)
    token = taken = without = 0

    def valid(i):
        return i if 0 <= i < num_blocks else -1

    for b in range(batch):
        c, n = max(int(ctx[b]), 0), max(int(new[b]), 0)
        n = min(n, 2**31 - 1 - c, max_tokens - token)
        have = min(-(-c // block_size), max_blocks)
        need = min(-(-(c + n) // block_size), max_blocks) if n else have
        for j in range(have, need):
            i = begin + taken
            tables[b, j] = valid(int(free_blocks[i])) if i < end else -1
            taken += 1
        start[b], kv[b] = token, c + n
        for i in range(n):
            p = c + i
            page = p // block_size
            block = valid(int(tables[b, page])) if page < max_blocks else -1
            pos[token] = p
            slots[token] = block * block_size + p % block_size if block >= 0 else -1
            without += block < 0
            token += 1
    start[batch] = token
    return tables, kv, start, pos, slots, np.array(
        [token, taken, without, max(begin, min(begin + taken, end))], np.int32)


def qk_norm_rope_f64(x, weight, cos, sin, positions, rot, interleaved, eps):
    """(y, size): x [tokens, heads, dim] normalised and rotated, and |a| + |b| of the pair that each
    value comes from (after the norm), the scale of its rounding errors."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    y, size, half = x.copy(), np.abs(x), rot // 2
    for j in range(half):
        i0, i1 = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        c = np.asarray(cos, np.float64)[positions, j][:, None]
        s = np.asarray(sin, np.float64)[positions, j][:, None]
        a, b = x[..., i0], x[..., i1]
        y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
        size[..., i0] = size[..., i1] = np.abs(a) + np.abs(b)
    return y, size


def quantise(x, group):
    """(codes u8 [..., dim], scale f16, offset f16 [..., dim / group])."""
    x = np.asarray(x, np.float64)
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // group, group))
    lo, hi = g.min(-1), g.max(-1)
    with np.errstate(all="ignore"):
        scale = np.minimum(((hi - lo) / 15.0).astype(np.float32), np.float32(65504)).astype(np.float16)
        offset = np.clip(lo, -65504, 65504).astype(np.float32).astype(np.float16)
        odd = ~np.isfinite(g).all(-1)
        scale[odd] = np.nan
        offset[odd] = np.nan
        s = scale.astype(np.float64)[..., None]
        q = np.rint((g - offset.astype(np.float64)[..., None]) / s)
    codes = np.where(s > 0, np.clip(np.nan_to_num(q), 0, 15), 0).astype(np.uint8)
    return codes.reshape(x.shape), scale, offset


def values_f64(codes, scale, offset):
    """code * scale + offset of codes [..., dim] and groups [..., dim / group]."""
    n = scale.shape[-1]
    c = codes.astype(np.float64).reshape(codes.shape[:-1] + (n, codes.shape[-1] // n))
    v = c * scale.astype(np.float64)[..., None] + offset.astype(np.float64)[..., None]
    return v.reshape(codes.shape)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(packed.shape[:-1] + (-1,))


def attention_f64(q, k, v, k_size, v_size, tables, kv_lens, query_start, scale, block_size):
    """(o, bound): q [tokens, q_heads, dim]; k, v f64 [block, kv_head, block_size, dim] dequantised,
    k_size, v_size the sizes code * scale + |offset| and (of centred codes) 8 * scale + |offset + 8 *
    scale| that their products are summed in.  Rows of no sequence are NaN.

    bound: what f32 sums of these products can be off by, for each output.  A score is a sum of
    magnitude A = |scale| sum |q| k_size whose terms are held to 2^-22 (two f16 halves) and summed
    in at most 16 steps that drop at most 2^-23 each: 2^-18 A.  A weight is then off by a factor
    1 + eta, eta = 2 * 2^-18 max A + 2^-20; the sums over n positions add n/16 + 16 such steps, to
    the numerator and the denominator."""
    q = np.asarray(q, np.float64)
    tokens, hq, d = q.shape
    blocks, hk = k.shape[:2]
    per = hq // hk
    o = np.full(q.shape, np.nan)
    bound = np.zeros(q.shape)
    batch, max_blocks = tables.shape
    if query_start is None:
        query_start = np.arange(batch + 1)
    for b in range(batch):
        t0, n = int(query_start[b]), int(query_start[b + 1] - query_start[b])
        kv = min(max(int(kv_lens[b]), 0), max_blocks * block_size)
        pos = np.arange(kv)
        page = tables[b, pos // block_size]
        there = (page >= 0) & (page < blocks)
        pos, page = pos[there], page[there]
        for h in range(hk if n else 0):
            ks, vs = k[page, h, pos % block_size], v[page, h, pos % block_size]
            kz, vz = k_size[page, h, pos % block_size], v_size[page, h, pos % block_size]
            for i in range(n):
                m = int((pos < int(kv_lens[b]) - n + i + 1).sum())
                rows = slice(h * per, (h + 1) * per)
                if m == 0:
                    o[t0 + i, rows] = 0
                    continue
                x = q[t0 + i, rows]
                s = scale * (x @ ks[:m].T)
                a = abs(scale) * (np.abs(x) @ kz[:m].T)
                w = np.exp(s - s.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                o[t0 + i, rows] = w @ vs[:m]
                eta = 2 * 2.0**-18 * a.max(-1, keepdims=True) + 2.0**-20
                bound[t0 + i, rows] = (w @ vz[:m]) * (np.expm1(2 * eta) + 2 * (m / 16 + 16) * 2.0**-23)
    return o, bound
