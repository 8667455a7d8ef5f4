"""Packed prompt attention at scores and values far apart, against the
definition in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200.context import CudaContext  # noqa: E402
from tests import _q8_cache as ref  # noqa: E402
from tests.test_gpu_attention_packed import attend  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


@pytest.mark.parametrize("hd,qh,kvh", [(64, 8, 2), (128, 4, 2)])
@pytest.mark.parametrize("order", ["first", "last", "mixed"])
@pytest.mark.parametrize("gap", [12, 16, 20, 26])
def test_little_weight_on_large_v(ctx, hd, qh, kvh, order, gap):
    """Half of the positions have 2^-gap of the others' weight and V of 6e4
    against 1e-3.  A probability keeps f16's 11 bits down to 2^-21 of the
    row's reference maximum, which is at most its maximum, and is off by at
    most 2^-32 of it below: over the attended positions at most 2^-32 times
    the sum of their |v|, as the sum of the probabilities is 1 or more in
    units of the maximum.  One query dimension alone is not zero, so a score
    is one exact product."""
    r = np.random.default_rng(gap + hd)
    n, tail = 400, 40
    part = np.arange(n) // 8 % 2 == 0 if order == "mixed" else np.arange(n) < n // 2
    if order == "last":
        part = ~part
    part[n - tail:] = False
    q, k = np.zeros((n, qh, hd)), r.normal(0, 1, (n, kvh, hd))
    q[:, :, 0] = 1.0
    k[:, :, 0] = r.uniform(-0.5, 0, (n, kvh)) - gap * part[:, None]
    v = r.uniform(0.5, 1.0, (n, kvh, hd)) * np.where(part, 6e4, 1e-3)[:, None, None]
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    got = attend(ctx, q, k, v, [0, n], [0, n], math.log(2.0))
    rows = np.arange(n - tail, n)
    want, mag = ref.attention(q[rows], k, v, rows + 1, math.log(2.0))
    below = 2.0 ** -32 * np.abs(v.astype(np.float64)).sum(0).repeat(qh // kvh, 0) \
        if gap > 20 else 0.0
    ref.check_attention(got[rows], want, mag, lost=below)
    assert ctx.device_status() == 0
