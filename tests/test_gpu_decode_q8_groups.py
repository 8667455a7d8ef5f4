"""Decode attention over the 8-bit cache with rows split over CTAs at every
kind of grouping, at a bound that leaves nothing for probabilities held in
few bits."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200.context import CudaContext  # noqa: E402
from tests import _q8_cache as ref  # noqa: E402
from tests.test_gpu_kv_cache_q8 import Cache, keys, starts_of  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


def run(ctx, lens, qh, kvh, hd, bt, seed, scale=None):
    """V of one sign and nearly one size, so that bits lost from the
    probabilities or in joining parts would show in the output."""
    r = np.random.default_rng(seed)
    c = Cache(ctx, lens, kvh, hd, bt, seed=seed)
    total = int(sum(lens))
    v = 2.0 + 0.1 * r.normal(0, 1, (total, kvh, hd))
    c.append(keys(r, total, kvh, hd), v.astype(np.float16), lens, starts_of(lens))
    q = r.normal(0, 1, (len(lens), qh, hd)).astype(np.float16)
    got = c.decode(q, lens, scale)
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        k, v = (ref.rows(c.host[m], c.scale[m], c.table[b], int(n)) for m in "kv")
        ref.check_attention(got[b:b + 1], *ref.attention(
            q[b:b + 1], k, v, [n], ref.default_scale(hd) if scale is None else scale), held=0.0)
    assert np.array_equal(got, c.decode(q, lens, scale))
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("qh,kvh", [(1, 1), (2, 1), (3, 1), (5, 1), (6, 2), (7, 1), (8, 1),
                                    (9, 1), (16, 1), (20, 2), (24, 2), (40, 1)])
def test_split_rows_of_any_grouping(ctx, hd, qh, kvh):
    """Rows of 47 to 282 units (24 and fewer are not split): parts of one to
    eight heads, of several head groups, joined from two and from many."""
    run(ctx, [3000], qh, kvh, hd, 64, seed=qh)
    run(ctx, [9013], qh, kvh, hd, 32, seed=qh + 1)
    run(ctx, [3500, 0, 5], qh, kvh, hd, 16, seed=qh + 2, scale=0.2)


@pytest.mark.parametrize("hd,qh,kvh", [(64, 32, 2), (128, 12, 4), (128, 10, 2), (64, 7, 1)])
def test_ragged_batch_of_split_rows(ctx, hd, qh, kvh):
    """More than 16 sequences, more rows than CTAs at 32/2 and 12/4 (equal
    shares that cut rows anywhere), fewer at the others."""
    r = np.random.default_rng(hd + qh)
    lens = r.integers(0, 1500, 60)
    lens[[3, 17, 40]] = [3000, 4100, 2777]
    run(ctx, lens.tolist(), qh, kvh, hd, 32, seed=qh)


@pytest.mark.parametrize("qh,kvh,hd,bt,lens", [
    (32, 8, 128, 16, [117]), (32, 8, 64, 32, [1, 15, 16, 17, 31, 33]), (5, 1, 64, 48, [500]),
    (21, 3, 128, 64, [200, 7]), (16, 1, 128, 256, [700]), (40, 2, 128, 32, [77])])
def test_short_rows(ctx, qh, kvh, hd, bt, lens):
    run(ctx, lens, qh, kvh, hd, bt, seed=hd + qh)


@pytest.mark.parametrize("hd,qh,kvh", [(64, 8, 2), (128, 5, 1)])
@pytest.mark.parametrize("n", [1, 2, 17, 48, 100])
def test_outputs_are_rounded_once(ctx, hd, qh, kvh, n):
    """Queries of zeros: every weight is 1 and every f32 step but the scales'
    products is exact or below 2^-18 of the sum (100 additions of 2^-24, a
    reciprocal and a product), so an output is the mean of V within half a
    step of f16 and 2^-17.  The rows of a block share their product, so a
    product held in 11 bits would be off by up to 2^-12 in all of them."""
    r = np.random.default_rng(n + hd)
    c = Cache(ctx, [n], kvh, hd, 16, seed=n)
    v = r.uniform(0.5, 1.0, (n, kvh, hd)).astype(np.float16)
    c.append(keys(r, n, kvh, hd), v, [n], [0, n])
    q = np.zeros((1, qh, hd), np.float16)
    got = c.decode(q, [n]).astype(np.float64)
    k, v = (ref.rows(c.host[m], c.scale[m], c.table[0], n) for m in "kv")
    want, mag = ref.attention(q, k, v, [n], 1.0)
    half = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64) / 2
    assert (np.abs(got - want) <= half + mag * 2.0 ** -17).all()


@pytest.mark.parametrize("batch", [31, 32, 33])
@pytest.mark.parametrize("top", [90, 2500])
def test_shares_found_by_warps_and_by_the_cta(ctx, batch, top):
    """Around the number of sequences up to which a warp finds its share alone,
    with short rows and with split ones, empty sequences at both ends."""
    r = np.random.default_rng(batch)
    lens = r.integers(0, top, batch)
    lens[[0, 5, batch - 1]] = 0
    lens[batch - 2] = 2 * top
    run(ctx, lens.tolist(), 4, 2, 64, 32, seed=batch)
    lens[batch - 1] = 7
    run(ctx, lens.tolist(), 8, 1, 128, 16, seed=batch)
