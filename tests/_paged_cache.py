"""The paged f16 cache for the tests: pages, their rows and attention over
them, written from the definitions."""
from __future__ import annotations

import numpy as np

from mote_b200.types import DType, plain
from tests import _q8_cache

KINDS = {np.dtype(np.float16): DType.F16, np.dtype(np.float32): DType.F32,
         np.dtype(np.int32): DType.I32}


def put(ctx, a):
    a = np.ascontiguousarray(a)
    return ctx.from_numpy(plain(a.shape, KINDS[a.dtype]), a)


def get(ctx, t, dtype=np.float16):
    return ctx.read_numpy(t, dtype)


def starts_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def tables_of(lens, block, rng, spare=3, width=None):
    """(block tables with -1 where unused, number of blocks): pages in no order."""
    need = [-(-int(n) // block) for n in lens]
    blocks = sum(need) + spare
    order = rng.permutation(blocks)
    table = np.full((len(need), max([1, *need]) if width is None else width), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, blocks


def rows(cache, table_row, length):
    """[length, kv_heads, head_dim]: the cached rows of one sequence."""
    block = cache.shape[2]
    blk = np.asarray(table_row[:-(-length // block)], np.int64)
    return cache[blk].transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], cache.shape[3])[:length]


def attention(q, k_cache, v_cache, table, starts, lens, scale):
    """(out, mean |v|) in 64 bits, zeros where nothing is attended."""
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    for b, n in enumerate(lens):
        s0, s1 = int(starts[b]), int(starts[b + 1])
        if s1 > s0:
            reach = int(n) - (s1 - s0) + 1 + np.arange(s1 - s0)
            k, v = rows(k_cache, table[b], int(n)), rows(v_cache, table[b], int(n))
            out[s0:s1], mag[s0:s1] = _q8_cache.attention(q[s0:s1], k, v, reach, scale)
    return out, mag


def rotated(x, cos, sin, interleaved):
    """rope_f32's operations on [tokens, heads, head_dim] f16, rounded to f16 once."""
    pairs = cos.shape[1]
    out = x.copy()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else \
        (slice(0, pairs), slice(pairs, 2 * pairs))
    xa, xb = x[..., a].astype(np.float32), x[..., b].astype(np.float32)
    c, s = cos[:, None], sin[:, None]
    out[..., a] = (xa * c - xb * s).astype(np.float16)
    out[..., b] = (xb * c + xa * s).astype(np.float16)
    return out


def append(k_cache, v_cache, table, starts, lens, k, v):
    """In place: the rows of every sequence become its last positions."""
    block = k_cache.shape[2]
    for b, n in enumerate(lens):
        s0, s1 = int(starts[b]), int(starts[b + 1])
        for t in range(s0, s1):
            p = int(n) - s1 + t
            k_cache[table[b, p // block], :, p % block] = k[t]
            v_cache[table[b, p // block], :, p % block] = v[t]
