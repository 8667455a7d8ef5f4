"""Packed prompt attention at scores of 24000 and more: equal scores weigh the same on
both sides of a new maximum.

Scores are exact by construction: q = (256, 1, c, 0 ...) and k = (96, s, 1, 0 ...)
give 24576 + s + c, a sum of multiples of 1/8 below 2^15."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200.context import CudaContext  # noqa: E402
from tests.test_gpu_attention_packed import attend, check  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


@pytest.mark.parametrize("hd", [64, 128])
def test_ties_on_both_sides_of_a_new_maximum(ctx, hd):
    """Two equal scores, between them the largest, for which the running maximum moves:
    7.93 in log2 units above the first score, then 8.66."""
    n, qh = 600, 4
    q, k, v = np.zeros((n, qh, hd)), np.zeros((n, 1, hd)), np.zeros((n, 1, hd))
    q[..., 0], q[..., 1] = 256, 1
    q[..., 2] = np.random.default_rng(hd).integers(0, 2048, (n, qh))
    k[..., 0], k[..., 1], k[..., 2] = 96, -64, 1
    for p, s in ((10, -5.5), (140, 0.0), (270, 0.5), (400, 0.0)):
        k[p, 0, 1] = s
    v[140], v[400] = 1, -1
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    check(attend(ctx, q, k, v, [0, n], [0, n], scale=1.0), q, k, v, [0, n], [0, n], scale=1.0)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_scores_around_the_bound(ctx, hd):
    """Rows side by side whose scores are s + c with c from -2047 to 2047: below and above
    2^10 in log2 units, of both signs, within a warp's rows."""
    n, qh = 600, 4
    q, k, v = np.zeros((n, qh, hd)), np.zeros((n, 1, hd)), np.zeros((n, 1, hd))
    q[..., 1], q[..., 2] = 1, np.random.default_rng(hd).integers(-2047, 2048, (n, qh))
    k[..., 1], k[..., 2] = -64, 1
    for p, s in ((10, -5.5), (140, 0.0), (270, 0.5), (400, 0.0), (500, 0.5)):
        k[p, 0, 1] = s
    v[140], v[400], v[270], v[500] = 1, -1, 0.25, -0.25
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    check(attend(ctx, q, k, v, [0, n], [0, n], scale=1.0), q, k, v, [0, n], [0, n], scale=1.0)
    assert ctx.device_status() == 0
