"""Paged attention at scores of 24000 and more, where 2^-24 of a score is as much
as a probability may be off: equal scores have to weigh the same wherever they
stand, in one row's tiles and in the parts that a long row is cut into.

Scores are exact by construction: q = (256, 1, c, 0 ...) and k = (96, s, 1, 0 ...)
give 24576 + s + c, a sum of multiples of 1/8 below 2^15."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200.context import CudaContext  # noqa: E402
from tests import _paged_cache as ref  # noqa: E402
from tests._q8_cache import check_attention  # noqa: E402
from tests.test_gpu_paged_attention import expected, inputs, run  # noqa: E402

FAR = -64.0  # e^-64 of the others


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


def exact(new, past, hd, scores, values):
    """One sequence, whose position p has the score scores.get(p, FAR) beside what is
    each query's own, and the value values.get(p, 0)."""
    t = inputs([new], [past], 4, 1, hd, 16, seed=new, unused=0)
    for name in ("q", "k_cache", "v_cache"):
        t[name][:] = 0
    t["q"][..., 0], t["q"][..., 1] = 256, 1
    t["q"][..., 2] = np.random.default_rng(past).integers(0, 2048, (new, 4))
    t["k_cache"][..., 0], t["k_cache"][..., 1], t["k_cache"][..., 2] = 96, FAR, 1
    for p, s in scores.items():
        t["k_cache"][t["table"][0, p // 16], 0, p % 16, 1] = s
    for p, v in values.items():
        t["v_cache"][t["table"][0, p // 16], 0, p % 16] = v
    return t


def verify(ctx, t):
    want, mag = expected(t, 1.0)
    check_attention(run(ctx, t, scale=1.0), want, mag)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past", [(1, 9000), (4, 9000), (5, 9000), (61, 9000), (200, 30000)])
def test_ties_in_parts_whose_references_differ(ctx, hd, new, past):
    """The largest score stands at two places far apart.  Before the first of them comes
    one that is 3 lower, from which a running maximum does not move for it."""
    verify(ctx, exact(new, past, hd, {10: -3.0, 200: 0.0, 7000: 0.0}, {200: 1.0, 7000: -1.0}))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 4, 5, 61, 200])
def test_ties_on_both_sides_of_a_new_maximum(ctx, hd, new):
    """Two equal scores, between them the largest, for which the running maximum moves:
    7.93 in log2 units above the first score, then 8.66."""
    verify(ctx, exact(new, 600, hd, {10: -5.5, 140: 0.0, 270: 0.5, 400: 0.0}, {140: 1.0, 400: -1.0}))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past", [(1, 9000), (4, 9000), (61, 9000), (200, 600)])
def test_scores_around_the_bound(ctx, hd, new, past):
    """Rows side by side whose scores are s + c with c from -2047 to 2047: below and above
    2^10 in log2 units, of both signs, within a warp's rows."""
    scores = {10: -5.5, 140: 0.0, 270: 0.5, 400: 0.0, past - 100: 0.5}
    t = exact(new, past, hd, scores, {140: 1.0, 270: 0.25, 400: -1.0, past - 100: -0.25})
    t["q"][..., 0] = 0
    t["q"][..., 2] = np.random.default_rng(new).integers(-2047, 2048, (new, 4))
    verify(ctx, t)
