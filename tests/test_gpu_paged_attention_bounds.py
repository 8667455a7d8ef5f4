"""Paged attention with a bound on the new tokens that is far above their number, and
with a workspace of exactly the size that is asked for."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200._native import lib  # noqa: E402
from mote_b200.context import CudaContext  # noqa: E402
from tests._paged_cache import get, put  # noqa: E402
from tests._q8_cache import check_attention  # noqa: E402
from tests.test_gpu_paged_attention import expected, hold, inputs, run, verify  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past", [([1], [3000]), ([3], [40]), ([4], [700]), ([1, 1], [5000, 40]),
                                      ([2, 1], [90, 0]), ([5], [600])])
def test_a_bound_beyond_the_rows_changes_nothing(ctx, hd, new, past):
    """No sequence has more tokens than q has rows, so a larger bound names the same
    kernels: the same bits."""
    t = inputs(new, past, 8, 2, hd, 16, seed=past[0])
    want = verify(ctx, t, most=sum(new))
    for most in (sum(new) + 1, 64, 1000, 1 << 30):
        np.testing.assert_array_equal(run(ctx, t, most).view(np.uint16), want.view(np.uint16))
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past,most", [
    ([1], [20000], 1), ([1] * 5, [9000, 0, 70, 3000, 20], 2),       # one set of columns
    ([4], [9000], 4), ([3, 4, 1], [5000, 9000, 0], 4),              # two
    ([61], [9000], 61), ([300, 1, 40, 1], [2000, 9000, 0, 30], 300)])  # chunks, and both kernels
def test_workspace_of_the_size_that_is_asked_for(ctx, hd, new, past, most):
    """Behind `bytes` nothing is written, the counters are left at zero, and the rest
    needs no initialisation."""
    t = inputs(new, past, 8, 2, hd, 32, seed=len(new), unused=0)
    need = ctypes.c_uint64(0)
    assert lib().mote_cuda_gqa_attention_paged_f16_workspace_bytes(8, 2, hd, most, ctypes.byref(need)) == 0
    size = need.value
    assert size > 768
    behind = 64 << 20  # more than the largest size, so that what passed the end would show here
    fill = np.full(size // 4 + behind // 4, 0x7fc00001, np.int32)
    fill[:192] = 0
    ws, held = put(ctx, fill), hold(ctx, t)
    ptrs = [held[n].pointer for n in ("q", "k_cache", "v_cache", "table", "starts", "lens", "out")]
    args = (*ptrs, sum(new), len(new), 8, 2, hd, t["k_cache"].shape[0], 32, t["table"].shape[1], most, 0.125)
    assert lib().mote_cuda_gqa_attention_paged_f16(*args, ws.pointer, size - 1, ctx.stream) == 1
    want, mag = expected(t, 0.125)
    for _ in range(2):
        ctx.upload_numpy(held["out"], np.zeros(t["q"].shape, np.float16))
        assert lib().mote_cuda_gqa_attention_paged_f16(*args, ws.pointer, size, ctx.stream) == 0
        check_attention(get(ctx, held["out"]), want, mag)
    after = get(ctx, ws, np.int32)
    assert size % 4 == 0 and (after[:192] == 0).all() and (after[size // 4:] == 0x7fc00001).all()
    assert ctx.device_status() == 0
