"""GPU parity of causal attention over packed prompts with the definition in
64 bits (bound: tests/_q8_cache.py ``check_attention``)."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200 import ops  # noqa: E402
from mote_b200.context import CudaContext  # noqa: E402
from mote_b200.types import DType, plain  # noqa: E402
from tests import _q8_cache as ref  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


def f16(ctx, a):
    a = np.ascontiguousarray(a, dtype=np.float16)
    return ctx.from_bytes(plain(a.shape, DType.F16), a)


def i32(ctx, a):
    a = np.ascontiguousarray(a, dtype=np.int32)
    return ctx.from_bytes(plain(a.shape, DType.I32), a)


def starts_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def attend(ctx, q, k, v, qs, ks, scale=None):
    out = f16(ctx, np.full(q.shape, 7.0))
    ops.gqa_attention_packed_f16(ctx, f16(ctx, q), f16(ctx, k), f16(ctx, v), i32(ctx, qs),
                                 i32(ctx, ks), out, scale)
    return np.frombuffer(ctx.read_bytes(out), np.float16).reshape(q.shape)


def check(got, q, k, v, qs, ks, scale=None, rows=None):
    """Every sequence, or `rows` (b, index) of it where all would take long."""
    scale = ref.default_scale(q.shape[2]) if scale is None else scale
    for b in range(len(qs) - 1):
        nq, nk = qs[b + 1] - qs[b], ks[b + 1] - ks[b]
        i = np.arange(nq) if rows is None or nq <= rows else \
            np.unique(np.linspace(0, nq - 1, rows).astype(int))
        kb, vb = k[ks[b]:ks[b + 1]], v[ks[b]:ks[b + 1]]
        want, mag = ref.attention(q[qs[b] + i], kb, vb, nk - nq + i + 1, scale)
        ref.check_attention(got[qs[b] + i], want, mag)


def inputs(seed, tokens, kv_tokens, qh, kvh, hd):
    r = np.random.default_rng(seed)
    return tuple(r.normal(0, 1, s).astype(np.float16)
                 for s in ((tokens, qh, hd), (kv_tokens, kvh, hd), (kv_tokens, kvh, hd)))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("qh,kvh,lens", [
    (32, 8, [1]), (32, 8, [23]), (4, 1, [31, 32, 33, 1, 0, 64]), (8, 8, [127, 128, 129]),
    (6, 2, [130, 5, 85]), (5, 1, [300]), (14, 2, [150, 0, 0, 37]), (32, 2, [100, 9]),
    (8, 1, [16, 257]), (24, 1, [70]), (128, 1, [12, 3]), (33, 1, [65])])
def test_whole_prompts(ctx, hd, qh, kvh, lens):
    s = starts_of(lens)
    q, k, v = inputs(qh + hd, sum(lens), sum(lens), qh, kvh, hd)
    check(attend(ctx, q, k, v, s, s), q, k, v, s, s)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("qh,kvh,nq,nk", [
    (8, 2, [5, 1, 64], [133, 700, 128]), (4, 4, [130], [257]), (32, 8, [1, 1, 1], [1, 500, 129]),
    (8, 2, [40, 9, 3], [7, 0, 3]), (3, 1, [200], [1]), (8, 2, [0, 6], [50, 20])])
def test_prompts_continued_and_rows_with_nothing(ctx, hd, qh, kvh, nq, nk):
    qs, ks = starts_of(nq), starts_of(nk)
    q, k, v = inputs(hd + sum(nk), sum(nq), sum(nk), qh, kvh, hd)
    got = attend(ctx, q, k, v, qs, ks, 0.2)
    check(got, q, k, v, qs, ks, 0.2)
    for b in range(len(nq)):  # before the first position: zeros
        assert (got[qs[b]:qs[b] + max(0, nq[b] - nk[b])] == 0).all()
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd,qh,kvh,lens", [(64, 8, 2, [2500, 300]), (128, 4, 1, [3333]),
                                            (128, 2, 2, [1500, 1, 900]), (64, 64, 8, [640])])
def test_long_prompts(ctx, hd, qh, kvh, lens):
    s = starts_of(lens)
    q, k, v = inputs(hd + qh, sum(lens), sum(lens), qh, kvh, hd)
    v = (v * 0.1 + 2).astype(np.float16)
    got = attend(ctx, q, k, v, s, s)
    check(got, q, k, v, s, s, rows=60)
    assert np.array_equal(got, attend(ctx, q, k, v, s, s))  # the same again


def test_many_short_sequences(ctx):
    r = np.random.default_rng(4)
    lens = r.integers(0, 20, 700)
    lens[100:140] = 0
    s = starts_of(lens)
    q, k, v = inputs(5, s[-1], s[-1], 4, 2, 64)
    check(attend(ctx, q, k, v, s, s), q, k, v, s, s)


def test_scores_that_grow_along_the_row(ctx):
    """The running maximum moves by far more than one tile's range."""
    n, hd = 900, 64
    q, k, v = inputs(6, n, n, 4, 1, hd)
    q = np.abs(q)
    k = (k * 0.05 + np.linspace(0, 3, n)[:, None, None]).astype(np.float16)
    s = [0, n]
    check(attend(ctx, q, k, v, s, s), q, k, v, s, s, rows=80)
    k = k[::-1].copy()
    check(attend(ctx, q, k, v, s, s), q, k, v, s, s, rows=80)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd,qh,kvh", [(64, 8, 2), (128, 4, 4), (128, 6, 2)])
def test_masked_places_do_not_reach_a_row(ctx, hd, qh, kvh, bad):
    """Another sequence's rows, later positions and rows of no sequence may
    hold anything: outputs before them are the same bits."""
    lens = [70, 1, 200, 40]
    s = starts_of(lens) + 3
    q, k, v = inputs(7, 330, 330, qh, kvh, hd)
    clean = attend(ctx, q, k, v, s, s)
    check(clean, q, k, v, s, s)
    assert (clean[:3] == 7).all() and (clean[s[-1]:] == 7).all()  # rows of no sequence
    q2, k2, v2 = q.copy(), k.copy(), v.copy()
    for x in (q2, k2, v2):
        x[:3] = bad
        x[s[-1]:] = bad
    assert np.array_equal(attend(ctx, q2, k2, v2, s, s), clean)
    # position 100 of the third sequence and all of the second
    at = s[2] + 100
    for i, x in enumerate((q2, k2, v2)):
        x[s[1]] = bad
        if i:
            x[at, 0, 5:9] = bad
    got = attend(ctx, q2, k2, v2, s, s)
    same = np.ones(330, bool)
    same[s[1]] = False
    same[at:s[3]] = False
    assert np.array_equal(got[same], clean[same])
    g = qh // kvh
    assert not np.isfinite(got[at:s[3], :g]).all(-1).any()
    assert np.array_equal(got[at:s[3], g:], clean[at:s[3], g:])  # the other heads


@pytest.mark.parametrize("hd", [64, 128])
def test_v_not_finite_where_it_is_attended(ctx, hd):
    """An infinity of V reaches exactly the rows and dimensions that attend it."""
    n = 300
    q, k, v = inputs(9, n, n, 4, 1, hd)
    v[130, 0, 3], v[280, 0, 7], v[281, 0, 9] = np.inf, -np.inf, np.nan
    got = attend(ctx, q, k, v, [0, n], [0, n])
    assert (got[130:, :, 3] == np.inf).all() and np.isfinite(got[:130]).all()
    assert (got[280:, :, 7] == -np.inf).all() and np.isfinite(got[:280, :, 7]).all()
    assert np.isnan(got[281:, :, 9]).all() and np.isfinite(got[:281, :, 9]).all()
    rest = np.setdiff1d(np.arange(hd), [3, 7, 9])
    want, mag = ref.attention(q, k, np.nan_to_num(v.astype(np.float64), posinf=0, neginf=0),
                              np.arange(n) + 1, ref.default_scale(hd))
    ref.check_attention(got[:, :, rest], want[:, :, rest], mag[:, :, rest])


def test_bad_offsets_skip_the_sequence(ctx):
    q, k, v = inputs(10, 60, 60, 4, 2, 64)
    good = [0, 20, 40, 60]
    clean = attend(ctx, q, k, v, good, good)
    for qs, ks, rows in (([0, 20, 40, 61], good, slice(0, 40)),
                         (good, [0, 20, 40, 61], slice(0, 40)),
                         ([-4, 20, 40, 60], good, slice(20, 60)),
                         (good, [0, 20, 10, 60], slice(0, 20))):
        got = attend(ctx, q, k, v, qs, ks)
        assert ctx.device_status() == 2
        assert np.array_equal(got[rows], clean[rows])
    attend(ctx, q, k, v, [0, 20, 10, 60], good)  # overlapping rows: told, whatever they hold
    assert ctx.device_status() == 2


def test_captured_and_replayed_with_other_lengths(ctx):
    """The offsets live on the device: one graph serves any lengths."""
    import torch

    q, k, v = inputs(11, 300, 300, 8, 2, 128)
    tq, tk, tv, to = (f16(ctx, a) for a in (q, k, v, np.zeros_like(q)))
    ts = i32(ctx, [0, 0, 0, 0])
    ops.gqa_attention_packed_f16(ctx, tq, tk, tv, ts, ts, to)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.ExternalStream(ctx.stream)
    with torch.cuda.graph(graph, stream=stream):
        ops.gqa_attention_packed_f16(ctx, tq, tk, tv, ts, ts, to)
    for s in ([0, 300, 300, 300], [0, 100, 101, 290], [7, 7, 150, 299]):
        s = np.array(s, np.int32)
        ctx.upload_numpy(ts, s)
        with torch.cuda.stream(stream):
            graph.replay()
        got = np.frombuffer(ctx.read_bytes(to), np.float16).reshape(q.shape)
        check(got, q, k, v, s, s, rows=40)
    del graph
    assert ctx.device_status() == 0


@pytest.mark.parametrize("batch,qh,kvh,hd", [(31, 8, 2, 64), (200, 4, 1, 64), (256, 4, 2, 128),
                                             (257, 2, 2, 64)])
def test_ragged_batches_with_cached_positions(ctx, batch, qh, kvh, hd):
    """Batches around the sizes where items are ranked another way: lengths
    from nothing to hundreds, some over cached positions, some with fewer
    positions than queries."""
    r = np.random.default_rng(batch)
    nq = r.integers(0, 60, batch)
    nq[r.integers(0, batch, 4)] = 400
    nk = np.maximum(0, nq + r.integers(-20, 200, batch))
    qs, ks = starts_of(nq), starts_of(nk)
    q, k, v = inputs(batch, qs[-1], ks[-1], qh, kvh, hd)
    check(attend(ctx, q, k, v, qs, ks), q, k, v, qs, ks, rows=12)
    assert ctx.device_status() == 0


def test_through_the_registry(ctx):
    from mote_b200 import kernel

    s = [0, 40, 100]
    q, k, v = inputs(12, 100, 100, 4, 2, 64)
    want = attend(ctx, q, k, v, s, s)
    runtime = kernel.Runtime()
    kernel.register_cuda_kernels(runtime.kernels_mut())
    entry = runtime.resolve(kernel.KernelKey("gqa_attention_packed", DType.F16), ctx.device)
    t = [f16(ctx, a) for a in (q, k, v)] + [i32(ctx, s), i32(ctx, s), f16(ctx, np.zeros_like(q))]
    entry.launch(ctx.device, kernel.KernelArgs((*(x.pointer for x in t), 100, 100, 2, 4, 2, 64,
                                                kernel.f32_bits(0.125), ctx.stream)))
    got = np.frombuffer(ctx.read_bytes(t[5]), np.float16).reshape(q.shape)
    assert np.array_equal(got, want)


def test_values_of_v_not_finite_before_a_long_prompt_end(ctx):
    """Infinities in tiles that every row of a later item sees in full, and in
    the rows behind a prompt whose length is a whole number of tiles."""
    n, hd = 512, 128
    q, k, v = inputs(13, n + 9, n + 9, 4, 2, hd)
    v[n:] = np.nan
    v[5, 1, 7] = -np.inf
    got = attend(ctx, q, k, v, [0, n], [0, n])
    assert (got[5:n, 2:, 7] == -np.inf).all() and np.isfinite(got[:n, :2]).all()
    assert np.isfinite(got[:5]).all() and (got[n:] == 7).all()
    ok = np.setdiff1d(np.arange(hd), [7])
    want, mag = ref.attention(q[:n], k[:n], np.nan_to_num(v[:n].astype(np.float64), neginf=0),
                              np.arange(n) + 1, ref.default_scale(hd))
    ref.check_attention(got[:n][..., ok], want[..., ok], mag[..., ok])
