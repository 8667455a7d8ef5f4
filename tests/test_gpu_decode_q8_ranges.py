"""Decode attention over the 8-bit cache where the sizes of V or of the
scores differ by many orders of magnitude, against the definition in 64 bits
over the cache's own values.  The bound leaves nothing for probabilities
(``held=0``): they are held to far below the output's rounding."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200.context import CudaContext  # noqa: E402
from tests import _q8_cache as ref  # noqa: E402
from tests.test_gpu_kv_cache_q8 import Cache  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


def check(c, got, q, lens, scale):
    for b, n in enumerate(lens):
        k, v = (ref.rows(c.host[m], c.scale[m], c.table[b], n) for m in "kv")
        ref.check_attention(got[b:b + 1], *ref.attention(q[b:b + 1], k, v, [n], scale), held=0.0)


@pytest.mark.parametrize("order", ["first", "last", "mixed"])
@pytest.mark.parametrize("big,small", [(65504, 2.0 ** -6), (6e4, 1e-3), (6e4, 1e-4), (1, 1)])
@pytest.mark.parametrize("hd,n", [(64, 1536), (128, 768), (128, 3000)])
def test_v_of_different_sizes(ctx, hd, n, big, small, order):
    """Positions of large V and little weight beside positions of small V that
    carry the weight: by regions that reach every warp, in both orders, and in
    turn every 16 positions.  Heads differ in how little the weight is, up to
    2^-36 and 2^-60.  One query dimension alone is not zero, so scores are one
    product and their f32 error at 60 log2 units is below 60 * 2^-23."""
    r = np.random.default_rng(n + hd)
    kvh, qh, bt = 2, 16, 16
    part = np.arange(n) // 16 % 2 == 0 if order == "mixed" else np.arange(n) < n // 2
    if order == "last":
        part = ~part
    for gap in (36.0, 60.0):
        k = r.normal(0, 0.2, (n, kvh, hd))
        k[:, :, 0] -= gap * part[:, None]
        v = r.uniform(0.5, 1.0, (n, kvh, hd)) * np.where(part, big, small)[:, None, None]
        v[128:144] = 0  # a block of scale 0
        q = np.zeros((1, qh, hd))
        q[0, :, 0] = np.arange(qh) % 8 / 8 + 0.125  # 1/8 to 1
        q = q.astype(np.float16)
        c = Cache(ctx, [n], kvh, hd, bt, seed=n)
        c.append(k.astype(np.float16), v.astype(np.float16), [n], [0, n])
        got = c.decode(q, [n], math.log(2.0))
        check(c, got, q, [n], math.log(2.0))
        assert np.array_equal(got, c.decode(q, [n], math.log(2.0)))
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd,n", [(64, 1536), (128, 3000)])
@pytest.mark.parametrize("spread", [5.0, 13.0, 40.0])
@pytest.mark.parametrize("sizes", [(0, 0), (-4, 0), (-14, 7), (5, 12)])
def test_scores_that_spread_widely(ctx, hd, n, spread, sizes):
    """Every step's largest weight is another power of two away, with V of
    ordinary sizes, of sizes that change from block to block, and of scales on
    both sides of 1.  Scores are one product, below 200 log2 units."""
    r = np.random.default_rng(n + int(spread))
    kvh, qh, bt = 2, 8, 16
    k = r.normal(0, 0.2, (n, kvh, hd))
    k[:, :, 0] = r.normal(0, spread, (n, kvh))
    size = 2.0 ** r.uniform(*sizes, -(-n // bt)).repeat(bt)[:n]
    v = r.uniform(0.5, 1.0, (n, kvh, hd)) * size[:, None, None]
    q = np.zeros((1, qh, hd))
    q[0, :, 0] = np.arange(qh) % 4 / 4 + 0.25
    q = q.astype(np.float16)
    c = Cache(ctx, [n], kvh, hd, bt, seed=n)
    c.append(k.astype(np.float16), v.astype(np.float16), [n], [0, n])
    check(c, c.decode(q, [n], math.log(2.0)), q, [n], math.log(2.0))
    assert ctx.device_status() == 0
