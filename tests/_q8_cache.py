"""The 8-bit KV cache's definition for the tests: appending, values and
attention in numpy, written from the formulas.

Scales and their reciprocals are f32 by definition; products of them with
f16 values and 8-bit integers are exact in 64 bits, so every rounding is the
one that the definition names and results compare bit for bit.
"""
from __future__ import annotations

import math

import numpy as np

NAN = np.float32(np.nan)


def append(cache, scales, table, x, lens_after, starts):
    """In place: rows x[starts[b]:starts[b + 1]] become the last positions."""
    bt = cache.shape[2]
    for b in range(len(lens_after)):
        rows = x[starts[b]:starts[b + 1]].astype(np.float64)
        pos = int(lens_after[b]) - len(rows)
        while len(rows):
            blk, off = table[b][pos // bt], pos % bt
            part, rows = rows[:bt - off], rows[bt - off:]
            for h in range(cache.shape[1]):
                old = np.float32(0) if off == 0 else scales[blk, h]
                xs = part[:, h]
                if np.isfinite(xs).all() and np.isfinite(old):
                    new = max(old, np.float32(np.abs(xs).max() / 127.0))
                    inv = np.float32(1) / new if new > 0 else np.float32(0)
                    if off and new != old:
                        ratio = np.float64(np.float32(old * inv))
                        cache[blk, h, :off] = np.rint(cache[blk, h, :off].astype(np.float64) * ratio)
                    cache[blk, h, off:off + len(xs)] = np.rint(xs * np.float64(inv))
                else:
                    new = NAN
                    cache[blk, h, :off + len(xs)] = 0
                scales[blk, h] = new
            pos += len(part)


def rows(cache, scales, table_row, length):
    """[length, kv_heads, head_dim] f32: the cached values of one sequence."""
    bt = cache.shape[2]
    blk = np.asarray(table_row[:-(-length // bt)], np.int64)
    v = cache[blk].astype(np.float32) * scales[blk][:, :, None, None]
    return v.transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], cache.shape[3])[:length]


def attention(q, k, v, reach, scale):
    """(out, mean |v|) in 64 bits: q [rows, q_heads, d] attends the first
    reach[row] of k, v [positions, kv_heads, d]; nothing attended: zeros."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    g = q.shape[1] // k.shape[1]
    out, mag = np.zeros_like(q), np.zeros_like(q)
    for i in range(len(q)):
        n = int(min(reach[i], len(k)))
        if n <= 0:
            continue
        for h in range(k.shape[1]):
            s = (q[i, h * g:(h + 1) * g] @ k[:n, h].T) * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[i, h * g:(h + 1) * g] = p @ v[:n, h]
            mag[i, h * g:(h + 1) * g] = p @ np.abs(v[:n, h])
    return out, mag


def check_attention(got, ref, mag, held=2.0 ** -11, lost=0.0):
    """f16 outputs against 64 bits.  Half a step of the output's own rounding
    (2^-11 of the value, 2^-25 below the normal range), half a step of each
    probability held in f16 (2^-11 of the weighted mean of |v|; `held` is 0
    for an operator that holds them in more), and 2^-13 of it for the f32
    steps: scores up to about 30 summed over 128 products are off by at most
    128 * 2^-24 * 30 = 2^-12.1 if every step rounds the same way and below
    2^-14 as roundings fall, exp2's approximation by 2^-22.  `lost` is what
    probabilities below the type's range may take from each output."""
    bound = np.abs(ref) * 2.0 ** -11 + mag * (held + 2.0 ** -13) + 2.0 ** -25 + lost
    off = np.abs(np.asarray(got, np.float64) - ref)
    assert np.isfinite(got).all()
    assert (off <= bound).all(), (off / bound).max()


def default_scale(head_dim):
    return 1.0 / math.sqrt(head_dim)
