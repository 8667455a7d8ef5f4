"""Decode attention over the 8-bit cache at scores whose own f32 steps are
larger than the range of exp2: equal scores have to weigh the same."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200.context import CudaContext  # noqa: E402
from tests import _q8_cache as ref  # noqa: E402
from tests.test_gpu_kv_cache_q8 import Cache  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


@pytest.mark.parametrize("hd,n", [(64, 1000), (128, 1000), (64, 4000)])
@pytest.mark.parametrize("low", [1.0, 0.5, -1.0])
def test_ties_at_vast_scores(ctx, hd, n, low):
    """Keys of one size, or of two in turn, so that each block has the same
    scale: scores up to 1e10 in log2 units, equal within each size (the same
    products in the same order) and apart by far more than exp2's range
    between them.  So the output is the mean of V over the larger."""
    r = np.random.default_rng(n)
    bt = 32
    k = np.full((n, 1, hd), 30000.0)
    k[1::2] *= low
    v = r.uniform(0.5, 1.0, (n, 1, hd))
    # sizes whose scores round up in f32 and sizes whose scores round down
    sizes = [30000, 27000, 65504, -3, -30000, 11000, -65504, 0.001, 900, -17000, 5000, 45000]
    c = Cache(ctx, [n], 1, hd, bt, seed=n)
    c.append(k.astype(np.float16), v.astype(np.float16), [n], [0, n])
    kk, vv = (ref.rows(c.host[m], c.scale[m], c.table[0], n) for m in "kv")
    for size in sizes:
        q = np.full((1, 1, hd), size).astype(np.float16)
        got = c.decode(q, [n])
        ref.check_attention(got, *ref.attention(q, kk, vv, [n], ref.default_scale(hd)), held=0.0)
    assert ctx.device_status() == 0
