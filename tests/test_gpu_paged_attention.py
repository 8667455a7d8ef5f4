"""Attention of new tokens over the paged f16 cache, against the definition in
64 bits: single tokens, drafted ones, chunks and mixes of them, and what their
masks, pages, splits and workspaces can go wrong at."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200 import ops  # noqa: E402
from mote_b200._native import lib  # noqa: E402
from mote_b200.context import CudaContext  # noqa: E402
from mote_b200.types import DType, plain  # noqa: E402
from tests import _paged_cache as ref  # noqa: E402
from tests._paged_cache import get, put  # noqa: E402
from tests import _q8_cache  # noqa: E402
from tests._q8_cache import check_attention  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


def inputs(new, past, qh, kvh, hd, block, seed, tail=0, unused=np.nan):
    """`tail`: rows behind the last sequence; `unused`: what the cache holds
    where no sequence has a position."""
    rng = np.random.default_rng(seed)
    new, past = np.asarray(new), np.asarray(past)
    lens, tokens = (new + past).astype(np.int32), int(new.sum()) + tail
    table, blocks = ref.tables_of(lens, block, rng)
    t = {"q": rng.normal(0, 1, (tokens, qh, hd)).astype(np.float16)}
    for name in ("k_cache", "v_cache"):
        c = rng.normal(0, 1, (blocks, kvh, block, hd)).astype(np.float16)
        live = np.zeros((blocks, block), bool)
        for b, n in enumerate(lens):
            for i in range(-(-int(n) // block)):
                live[table[b, i], :min(block, int(n) - i * block)] = True
        c.transpose(0, 2, 1, 3)[~live] = unused
        t[name] = c
    return t | {"table": table, "starts": ref.starts_of(new), "lens": lens}


def launch(ctx, held, most, scale=None):
    ops.gqa_attention_paged_f16(ctx, held["q"], held["k_cache"], held["v_cache"], held["table"],
                                held["starts"], held["lens"], held["out"], most, scale)


def hold(ctx, t, fill=7.0):
    held = {n: put(ctx, a) for n, a in t.items()}
    held["out"] = put(ctx, np.full(t["q"].shape, fill, np.float16))
    return held


def run(ctx, t, most=None, scale=None, fill=7.0):
    held = hold(ctx, t, fill)
    most = int(np.diff(t["starts"]).max()) if most is None else most
    launch(ctx, held, most, scale)
    return get(ctx, held["out"])


def expected(t, scale=None):
    scale = 1 / math.sqrt(t["q"].shape[-1]) if scale is None else scale
    return ref.attention(*(t[n] for n in ("q", "k_cache", "v_cache", "table", "starts", "lens")), scale)


def verify(ctx, t, most=None, scale=None):
    got = run(ctx, t, most, scale)
    n = int(t["starts"][-1])
    want, mag = expected(t, scale)
    check_attention(got[:n], want[:n], mag[:n])
    assert (got[n:] == 7.0).all()
    assert ctx.device_status() == 0
    return got


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 1000, 5003])
def test_one_token(ctx, hd, length):
    verify(ctx, inputs([1], [length - 1], 8, 2, hd, 16, seed=length))


@pytest.mark.parametrize("qh,kvh", [(1, 1), (2, 1), (3, 1), (10, 2), (7, 1), (16, 2), (9, 1),
                                    (32, 2), (17, 1), (32, 1), (40, 1), (128, 1), (24, 8), (8, 8)])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_groupings(ctx, qh, kvh, new):
    verify(ctx, inputs([new, 1, new], [300, 77, 0], qh, kvh, 64 if qh % 2 else 128, 32, seed=qh + new))


@pytest.mark.parametrize("block", [16, 32, 48, 64, 80, 96, 128, 144, 192, 240, 256])
@pytest.mark.parametrize("new", [1, 5, 100])
def test_pages(ctx, block, new):
    """Blocks that end inside a tile and tiles that end inside a block."""
    verify(ctx, inputs([new, 1, new], [700, 383, 2 * block - new % 7], 8, 2, 128, block, seed=block))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past", [
    ([2], [0]), ([4], [13]), ([8], [1000]), ([9], [119]), ([16], [112]), ([17], [0]), ([33], [95]),
    ([64], [64]), ([65], [1]), ([127], [0]), ([128], [128]), ([129], [1]), ([257], [700]),
    ([600], [0]), ([1000], [1500])])
def test_chunks(ctx, hd, new, past):
    verify(ctx, inputs(new, past, 8, 2, hd, 32, seed=new[0]))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past", [
    ([1, 1, 1, 1], [0, 5000, 17, 300]), ([3, 1, 8, 0, 2], [200, 0, 31, 90, 0]),
    ([1] * 40, list(range(0, 4000, 100))), ([200, 1, 1, 7, 1, 90], [300, 900, 0, 64, 2000, 0]),
    ([0, 0, 5, 0], [3, 0, 40, 16]), ([64, 64, 64], [0, 1000, 64]), ([1, 500, 1], [2500, 100, 2600]),
    ([2] * 70, [(37 * i) % 500 for i in range(70)]), ([20] * 33, [(61 * i) % 300 for i in range(33)])])
def test_mixed_batches(ctx, hd, new, past):
    verify(ctx, inputs(new, past, 8, 2, hd, 16, seed=len(new)))


@pytest.mark.parametrize("hd,qh,kvh,new,past", [
    (128, 8, 2, [1], [20000]), (64, 8, 2, [1], [20001]), (128, 8, 2, [4], [9000]),
    (128, 16, 2, [61], [9000]), (64, 4, 4, [130], [8000]), (128, 32, 1, [1], [12000]),
    (128, 8, 1, [1, 33, 2], [6000, 7000, 6500])])
def test_long_rows_are_split(ctx, hd, qh, kvh, new, past):
    """Rows over many CTAs, whose parts are joined; twice the same bits."""
    t = inputs(new, past, qh, kvh, hd, 64, seed=past[0])
    a = verify(ctx, t)
    np.testing.assert_array_equal(a.view(np.uint16), run(ctx, t).view(np.uint16))


@pytest.mark.parametrize("new,past", [([1, 1], [5, 40]), ([3, 2], [20, 0]), ([90, 40], [100, 0])])
def test_most_tokens_may_be_more_than_there_are(ctx, new, past):
    """The count that the host gives is a bound: a larger one gives the same
    values to rounding (another variant may run)."""
    t = inputs(new, past, 8, 2, 64, 16, seed=4)
    for most in (max(new), max(new) + 1, 17, 64, 1000, 1 << 30):
        if most >= max(new):
            verify(ctx, t, most=most)


def test_queries_before_the_first_position_get_zeros(ctx):
    """More new tokens than positions: rows without any are zeros, the others
    attend what there is."""
    for new, length in ((5, 3), (5, 0), (2, 1), (40, 7), (70, 0), (200, 130)):
        t = inputs([new, 3], [0, 20], 8, 2, 64, 16, seed=new)
        t["lens"][0] = length
        for name in ("k_cache", "v_cache"):
            t[name][np.isnan(t[name])] = 0
        got = verify(ctx, t)
        assert (got[:max(0, new - length)] == 0).all()


@pytest.mark.parametrize("new", [[1, 1], [3, 1], [50, 1]])
def test_rows_behind_the_last_sequence_keep_their_values(ctx, new):
    verify(ctx, inputs(new, [30, 9], 8, 2, 64, 16, seed=1, tail=9))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new,past", [([1], [18]), ([5], [28]), ([12], [0]), ([90], [64]), ([300], [10])])
@pytest.mark.parametrize("hd", [64, 128])
def test_what_is_masked_does_not_reach_a_row(ctx, bad, new, past, hd):
    """Later positions and what lies behind the last one hold infinities or
    NaN: rows that do not attend them are as without, rows that do show them."""
    t = inputs(new, past, 8, 2, hd, 32, seed=new[0], unused=bad)
    length = new[0] + past[0]
    clean, mag = expected(t)
    spoilt = {n: a.copy() for n, a in t.items()}
    at = past[0] + new[0] // 2  # a position that some rows attend
    spoilt["v_cache"][t["table"][0, at // 32], 0, at % 32, 3] = bad
    if new[0] > 1:
        spoilt["k_cache"][t["table"][0, (length - 1) // 32], 1, (length - 1) % 32] = bad
    got = run(ctx, spoilt)
    rows = np.arange(new[0]) + past[0]
    low = rows < at  # head 0 to 3: KV head 0
    check_attention(got[low][:, :4], clean[low][:, :4], mag[low][:, :4])
    cols = [c for c in range(hd) if c != 3]
    check_attention(got[:, :4][..., cols], clean[:, :4][..., cols], mag[:, :4][..., cols])
    shown = got[~low][:, :4, 3]
    assert (np.isnan(shown) if np.isnan(bad) else shown == bad).all()
    if new[0] > 1:
        check_attention(got[:-1, 4:], clean[:-1, 4:], mag[:-1, 4:])
    assert ctx.device_status() == 0


@pytest.mark.parametrize("new", [[1], [4], [70]])
@pytest.mark.parametrize("size", [1e-3, 30.0, 3e3, 6e4])
def test_scores_and_values_of_any_size(ctx, new, size):
    """Scores up to 6e4 and values up to 6e4; equal keys weigh the same."""
    t = inputs(new, [200], 4, 2, 64, 16, seed=2, unused=0)
    rng = np.random.default_rng(5)
    key = rng.normal(0, 1, 64)
    t["q"][:] = (key / np.linalg.norm(key)).astype(np.float16)
    t["k_cache"][:] = (key / np.linalg.norm(key) * min(size, 100)).astype(np.float16)
    t["v_cache"] = (rng.uniform(-1, 1, t["v_cache"].shape) * min(size, 6e4)).astype(np.float16)
    scale = max(1.0, size / 100)
    want, mag = expected(t, scale)
    check_attention(run(ctx, t, scale=scale), want, mag)


@pytest.mark.parametrize("new", [[1], [4], [70]])
def test_rising_scores(ctx, new):
    """Every tile's maximum is far above the one before."""
    t = inputs(new, [900], 4, 2, 128, 32, seed=3, unused=0)
    order = ref.rows(np.arange(t["k_cache"].size).reshape(t["k_cache"].shape), t["table"][0], 900 + new[0])
    flat = t["k_cache"].reshape(-1)
    flat[order] = (np.linspace(-3, 3, len(order))[:, None, None] * np.ones(order.shape)).astype(np.float16)
    t["q"][:] = np.abs(t["q"])
    want, mag = expected(t, 0.3)
    # scores of up to 128 * 3 * 0.3 * 0.8 = 92 on sums of one sign: each of 128
    # f32 steps may be off by half a step of that, 92 * 2^-24 * sqrt(128) rms
    check_attention(run(ctx, t, scale=0.3), want, mag, lost=mag * 2.0 ** -12)


@pytest.mark.parametrize("what", ["length below zero", "length past the table", "starts fall",
                                  "starts past the rows", "too many new", "starts below"])
@pytest.mark.parametrize("new", [[2, 1, 3], [40, 30, 50], [1, 60, 1]])
def test_sequences_out_of_range_are_skipped(ctx, what, new):
    t = inputs(new, [20, 40, 60], 8, 2, 64, 16, seed=6, unused=0)
    want, mag = expected(t)
    most, skipped = max(new), [1]
    if what == "length below zero":
        t["lens"][1] = -1
    elif what == "length past the table":
        t["lens"][1] = 16 * t["table"].shape[1] + 1
    elif what == "starts fall":
        t["starts"][1], t["starts"][2] = t["starts"][2], t["starts"][1] - 1
        skipped = None
    elif what == "starts past the rows":
        t["starts"][3] += 1
        skipped = [2]
    elif what == "starts below":
        t["starts"][0] = -1
        skipped = [0]
    else:
        most -= 1
        skipped = [b for b in range(3) if new[b] == max(new)]
    got = run(ctx, t, most)
    assert ctx.device_status() & 2
    if skipped is None:
        return
    starts = ref.starts_of(new)
    for b in range(3):
        rows = slice(starts[b], starts[b + 1])
        if b in skipped:
            assert (got[rows] == 7.0).all()
        else:
            check_attention(got[rows], want[rows], mag[rows])


@pytest.mark.parametrize("number", [-1, -7, 1 << 30, None])
@pytest.mark.parametrize("new", [[2, 1], [50, 1]])
def test_blocks_out_of_range_read_as_zeros(ctx, number, new):
    t = inputs(new, [100, 40], 8, 2, 64, 16, seed=7, unused=0)
    zeroed = {n: a.copy() for n, a in t.items()}
    for name in ("k_cache", "v_cache"):
        zeroed[name][t["table"][0, 2]] = 0
    want, mag = expected(zeroed)
    t["table"][0, 2] = len(t["k_cache"]) if number is None else number
    got = run(ctx, t)
    assert ctx.device_status() & 2
    check_attention(got, want, mag)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch,kinds", [(45, (1, 50)), (300, (1, 2, 9)), (700, (1, 0, 17)), (1000, (1,))])
def test_many_sequences(ctx, hd, batch, kinds):
    """More sequences than a warp's lanes, than a CTA's threads; of both kernels."""
    new = [kinds[i % len(kinds)] for i in range(batch)]
    verify(ctx, inputs(new, [(37 * i) % 130 for i in range(batch)], 4, 2, hd, 16, seed=batch))


@pytest.mark.parametrize("new", [[1, 1], [40, 1], [70, 90]])
def test_rows_before_the_first_sequence_keep_their_values(ctx, new):
    t = inputs(new, [30, 9], 8, 2, 64, 16, seed=2, unused=0)
    want, mag = expected(t)
    t["q"] = np.concatenate([np.repeat(t["q"][:1], 5, 0), t["q"]])
    t["starts"] = t["starts"] + 5
    got = run(ctx, t, max(new))
    assert (got[:5] == 7.0).all()
    check_attention(got[5:], want, mag)


@pytest.mark.parametrize("new", [[1], [3], [90]])
def test_a_query_of_nan_or_infinity_is_its_own(ctx, new):
    t = inputs(new, [200], 8, 2, 64, 16, seed=3, unused=0)
    want, mag = expected(t)
    t["q"][0, 1], t["q"][0, 6, 3] = np.nan, np.inf
    got = run(ctx, t).copy()
    assert np.isnan(got[0, 1]).all() and np.isnan(got[0, 6]).any()
    for name in (got, want, mag):
        name[0, [1, 6]] = 0
    check_attention(got, want, mag)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,past", [([1], [40]), ([3], [5000]), ([90], [20]), ([40], [9000]), ([50, 1], [4000, 80])])
def test_scores_of_minus_infinity_alone_are_no_mask(ctx, hd, new, past):
    """Positions are attended whose scores are all -infinity: 0 / 0, and not the zeros
    of a query that attends nothing.  A finite score among them takes it all."""
    t = inputs(new, past, 4, 1, hd, 16, 41, unused=0.0)
    t["q"][:] = 1.0
    t["k_cache"][..., 0] = -np.inf
    assert np.isnan(run(ctx, t)).all()
    for b, n in enumerate(t["lens"]):  # position 2 of each sequence
        t["k_cache"][t["table"][b, 0], :, 2] = 0.5
    got = run(ctx, t)
    for b, n in enumerate(t["lens"]):
        rows = got[t["starts"][b]:t["starts"][b + 1]]
        assert (rows == t["v_cache"][t["table"][b, 0], 0, 2]).all()


def test_positions_up_to_two_to_the_31st(ctx):
    """A length whose last unit of positions ends at 2^31, all pages one block.  Scores
    of -20 everywhere: positions behind the last one, had they weight e^0, would be
    four times as heavy as all of the sequence.  Weights are equal, so the result is
    the mean of V, here 1."""
    length = 0x7ffffff0
    t = {"q": put(ctx, np.full((1, 1, 64), 1.0, np.float16)),
         "k_cache": put(ctx, np.full((1, 1, 16, 64), -2.5, np.float16)),
         "v_cache": put(ctx, np.full((1, 1, 16, 64), 1.0, np.float16)),
         "table": put(ctx, np.zeros((1, length // 16), np.int32)),
         "starts": put(ctx, np.array([0, 1], np.int32)),
         "lens": put(ctx, np.array([length], np.int32)),
         "out": put(ctx, np.zeros((1, 1, 64), np.float16))}
    launch(ctx, t, 1)  # -2.5 * 64 / 8 = -20
    assert (get(ctx, t["out"]) == 1.0).all()


def test_offsets_past_32_bits(ctx):
    """Caches of more than 2^32 values: rows in the last blocks."""
    kvh, block, hd = 8, 256, 128
    blocks = (1 << 32) // (kvh * block * hd) + 5
    cache = [ctx.empty(plain((blocks, kvh, block, hd), DType.F16)) for _ in range(2)]
    rng = np.random.default_rng(4)
    for new, qh in (([300, 270], 16), ([1, 1], 16), ([40, 1], 16)):
        tokens, total = sum(new), 300
        t = {"qkv": rng.normal(0, 1, (600, qh + 2 * kvh, hd)).astype(np.float16),
             "cos": np.ones((600, 64), np.float32), "sin": np.zeros((600, 64), np.float32),
             "q_out": np.zeros((600, qh, hd), np.float16)}
        table = np.array([[blocks - 1, blocks - 4], [blocks - 2, blocks - 3]], np.int32)
        lens = np.array([total, total], np.int32)
        held = {n: put(ctx, a) for n, a in t.items()}
        tb, ln = put(ctx, table), put(ctx, lens)
        ops.rope_kv_cache_append_paged_f16(ctx, held["qkv"], held["cos"], held["sin"], held["q_out"],
                                           *cache, tb, put(ctx, np.array([0, 300, 600], np.int32)), ln)
        starts = ref.starts_of(new)
        q = rng.normal(0, 1, (tokens, qh, hd)).astype(np.float16)
        out = put(ctx, np.zeros(q.shape, np.float16))
        ops.gqa_attention_paged_f16(ctx, put(ctx, q), *cache, tb, put(ctx, starts), ln, out, max(new))
        got = get(ctx, out)
        for b in range(2):
            k, v = (t["qkv"][300 * b:300 * b + 300, qh + i * kvh:qh + (i + 1) * kvh] for i in range(2))
            rows = slice(starts[b], starts[b + 1])
            want, mag = _q8_cache.attention(q[rows], k, v, total - new[b] + 1 + np.arange(new[b]),
                                            1 / math.sqrt(hd))
            check_attention(got[rows], want, mag)
    assert ctx.device_status() == 0


def test_calls_of_two_contexts_at_once(ctx):
    """Two contexts' streams run the operators side by side."""
    cases = []
    for c in (ctx, CudaContext(0)):
        for new, past in (([61, 1], [3000, 900]), ([1] * 7, [4000, 1, 90, 700, 0, 33, 2000])):
            t = inputs(new, past, 8, 2, 128, 32, seed=len(new), unused=0)
            cases.append((c, t, hold(c, t), max(new)))
            launch(c, cases[-1][2], max(new))
    for _ in range(20):
        for c, _, held, most in cases:
            launch(c, held, most)
    for c, t, held, _ in cases:
        want, mag = expected(t)
        check_attention(get(c, held["out"]), want, mag)
        assert c.device_status() == 0


def test_graphs_that_share_the_workspace_take_turns(ctx):
    """Captured calls of several shapes and eager ones use one workspace, one
    after another; lengths are advanced between replays."""
    import torch

    shapes = [([1], [9000]), ([61, 1], [9000, 30]), ([1] * 5, [10, 700, 90, 0, 3000])]
    cases = []
    for new, past in shapes:
        t = inputs(new, past, 8, 2, 128, 64, seed=len(new), unused=0)
        held = hold(ctx, t)
        launch(ctx, held, max(new))
        cases.append((t, held, max(new)))
    stream, graphs = torch.cuda.ExternalStream(ctx.stream), []
    ctx.sync()
    for t, held, most in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream, capture_error_mode="relaxed"):
            launch(ctx, held, most)
    for shift in (0, 3, 7):
        for (t, held, most), graph in zip(cases, graphs):
            lens = (t["lens"] - shift).clip(0)
            ctx.upload_numpy(held["lens"], lens)
            with torch.cuda.stream(stream):
                graph.replay()
            ctx.sync()
            n = int(t["starts"][-1])
            want, mag = expected(t | {"lens": lens})
            check_attention(get(ctx, held["out"])[:n], want[:n], mag[:n])
    del graphs


def test_workspace_is_asked_for(ctx):
    """A call without its workspace, or with one that is too small, is refused."""
    import ctypes

    t = inputs([1], [40], 8, 2, 64, 16, seed=8)
    held = hold(ctx, t)
    ptrs = [held[n].pointer for n in ("q", "k_cache", "v_cache", "table", "starts", "lens", "out")]
    need = ctypes.c_uint64(0)
    for most in (1, 100):
        assert lib().mote_cuda_gqa_attention_paged_f16_workspace_bytes(8, 2, 64, most, ctypes.byref(need)) == 0
        args = (*ptrs, 1, 1, 8, 2, 64, t["k_cache"].shape[0], 16, t["table"].shape[1], most, 0.125)
        if need.value:
            assert lib().mote_cuda_gqa_attention_paged_f16(*args, None, 0, ctx.stream) == 1
            ws = ctx.empty(plain((need.value,), DType.U8))
            assert lib().mote_cuda_gqa_attention_paged_f16(*args, ws.pointer, need.value - 1, ctx.stream) == 1


def test_another_context(ctx):
    """Tensors of another context are refused, and each has its own workspace."""
    from mote_b200 import errors

    other = CudaContext(0)
    t = inputs([1, 50], [400, 30], 8, 2, 64, 16, seed=9)
    a, b = verify(ctx, t), verify(other, t)
    np.testing.assert_array_equal(a.view(np.uint16), b.view(np.uint16))
    held = hold(other, t)
    with pytest.raises(errors.WrongStorage):
        launch(ctx, held, 50)


def test_a_serving_run(ctx):
    """Tables, rotation and append, attention: prompts with pictures in chunks,
    then tokens one by one from a captured graph, against dense attention over
    the rotated rows in 64 bits."""
    import torch

    from mote_b200.types import RopeAxes

    qh, kvh, hd, block, batch = 8, 2, 128, 16, 3
    sections, theta = (16, 24, 24), 1e6
    rng = np.random.default_rng(12)
    steps = [[37, 5, 130], [20, 60, 1], [1, 1, 200], *[[1, 1, 1]] * 4]
    total = np.sum(steps, 0)
    table, blocks = ref.tables_of(total, block, rng)
    cache = {n: put(ctx, np.full((blocks, kvh, block, hd), np.nan, np.float16)) for n in "kv"}
    tables = put(ctx, table)
    seen = [{"k": [], "v": []} for _ in range(batch)]
    length = np.zeros(batch, np.int64)
    graph = held = None
    stream = torch.cuda.ExternalStream(ctx.stream)
    for step in steps:
        tokens = sum(step)
        positions = rng.integers(0, 500, (3, tokens)).astype(np.int32)
        qkv = rng.normal(0, 1, (tokens, qh + 2 * kvh, hd)).astype(np.float16)
        length = length + step
        fresh = {"positions": positions, "cos": np.zeros((tokens, 64), np.float32),
                 "sin": np.zeros((tokens, 64), np.float32), "qkv": qkv,
                 "q": np.zeros((tokens, qh, hd), np.float16), "starts": ref.starts_of(step),
                 "lens": length.astype(np.int32), "out": np.zeros((tokens, qh, hd), np.float16)}

        def layer():
            ops.rope_cos_sin_axes_f32(ctx, held["positions"], held["cos"], held["sin"], sections,
                                      theta, RopeAxes.Sections)
            ops.rope_kv_cache_append_paged_f16(ctx, held["qkv"], held["cos"], held["sin"], held["q"],
                                               cache["k"], cache["v"], tables, held["starts"],
                                               held["lens"], check=False)
            ops.gqa_attention_paged_f16(ctx, held["q"], cache["k"], cache["v"], tables,
                                        held["starts"], held["lens"], held["out"], max(step))

        if graph is not None and step == [1, 1, 1]:
            for n in ("positions", "qkv", "lens"):
                ctx.upload_numpy(held[n], fresh[n])
            with torch.cuda.stream(stream):
                graph.replay()
        else:
            held = {n: put(ctx, a) for n, a in fresh.items()}
            layer()
            if step == [1, 1, 1]:
                ctx.sync()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
                    layer()
                with torch.cuda.stream(stream):
                    graph.replay()
        ctx.sync()
        assert ctx.device_status() == 0
        # the definition, from the tables that the device made
        cos, sin = get(ctx, held["cos"], np.float32), get(ctx, held["sin"], np.float32)
        x = ref.rotated(qkv[:, :qh + kvh], cos, sin, False)
        starts = ref.starts_of(step)
        for b in range(batch):
            s = slice(starts[b], starts[b + 1])
            seen[b]["k"].append(x[s, qh:])
            seen[b]["v"].append(qkv[s, qh + kvh:])
            k, v = (np.concatenate(seen[b][n]) for n in "kv")
            want, mag = _q8_cache.attention(x[s, :qh], k, v, length[b] - step[b] + 1 + np.arange(step[b]),
                                            1 / math.sqrt(hd))
            check_attention(get(ctx, held["out"])[s], want, mag)
    del graph
