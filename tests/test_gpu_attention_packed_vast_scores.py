"""Packed prompt attention at scores whose own f32 steps are larger than the
range of exp2: equal scores have to weigh the same, and nothing overflows."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200.context import CudaContext  # noqa: E402
from tests.test_gpu_attention_packed import attend, check, starts_of  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("top", [100.0, 30000.0, 65504.0])
@pytest.mark.parametrize("low", [1.0, 0.5, -1.0])
def test_ties_at_vast_scores(ctx, hd, top, low):
    """Keys of one size, or of two in turn: scores up to 1e11 in log2 units,
    equal within each size and apart by far more than exp2's range between
    them, so the output is the mean of V over the larger."""
    r = np.random.default_rng(hd)
    lens = [300, 1, 37]
    s = starts_of(lens)
    k = np.full((s[-1], 2, hd), top)
    k[1::2] *= low
    q = np.full((s[-1], 8, hd), top)
    q[:, 1::2] = -3.0  # other heads prefer the lower keys, at smaller scores
    q[:, 2::4] = 0.001
    v = r.uniform(0.5, 1.0, k.shape)
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    check(attend(ctx, q, k, v, s, s), q, k, v, s, s)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("size", [30.0, 1000.0, 20000.0])
def test_random_at_vast_scores(ctx, size):
    """Random queries and keys of large size: one position has all the weight
    (scores of a row are apart by far more than their f32 error), so each
    output is a row of V."""
    r = np.random.default_rng(int(size))
    n, qh, kvh, hd = 300, 4, 2, 64
    q = np.zeros((n, qh, hd))
    q[:, :, 0] = size * r.choice([-1, 1], (n, qh))
    k = np.clip(r.normal(0, 1, (n, kvh, hd)) * size, -65504, 65504)
    k[:, :, 0] = np.stack([r.permutation(n) - n / 2 for _ in range(kvh)], 1) * size / n * 2
    v = r.normal(0, 1, (n, kvh, hd))
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    check(attend(ctx, q, k, v, [0, n], [0, n]), q, k, v, [0, n], [0, n])
    assert ctx.device_status() == 0
