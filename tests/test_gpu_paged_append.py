"""Rotation and append to the paged f16 cache: bit for bit against the
definition (rope_f32's operations and copies)."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200 import errors, ops  # noqa: E402
from mote_b200._native import lib  # noqa: E402
from mote_b200.context import CudaContext  # noqa: E402
from mote_b200.types import DType, RopeLayout, plain  # noqa: E402
from tests import _paged_cache as ref  # noqa: E402
from tests._paged_cache import get, put  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


def inputs(new, past, qh, kvh, hd, pairs, block, seed, tail=0):
    """`tail`: rows behind the last sequence."""
    rng = np.random.default_rng(seed)
    new, past = np.asarray(new), np.asarray(past)
    tokens = int(new.sum()) + tail
    table, blocks = ref.tables_of(new + past, block, rng)
    angle = rng.uniform(-4, 4, (tokens, pairs))
    return {"qkv": rng.normal(0, 1, (tokens, qh + 2 * kvh, hd)).astype(np.float16),
            "cos": np.cos(angle).astype(np.float32), "sin": np.sin(angle).astype(np.float32),
            "q_out": rng.normal(0, 1, (tokens, qh, hd)).astype(np.float16),
            "k_cache": rng.normal(0, 1, (blocks, kvh, block, hd)).astype(np.float16),
            "v_cache": rng.normal(0, 1, (blocks, kvh, block, hd)).astype(np.float16),
            "table": table, "starts": ref.starts_of(new), "lens": (new + past).astype(np.int32)}


def run(ctx, t, layout=RopeLayout.HalfSplit, **kw):
    held = {n: put(ctx, a) for n, a in t.items()}
    ops.rope_kv_cache_append_paged_f16(ctx, *held.values(), layout, **kw)
    return tuple(get(ctx, held[n]) for n in ("q_out", "k_cache", "v_cache"))


def expected(t, layout=RopeLayout.HalfSplit):
    qh, kvh = t["q_out"].shape[1], t["k_cache"].shape[1]
    q, k, v = t["q_out"].copy(), t["k_cache"].copy(), t["v_cache"].copy()
    x = ref.rotated(t["qkv"][:, :qh + kvh], t["cos"], t["sin"], layout is RopeLayout.Interleaved)
    n = int(t["starts"][-1])
    q[:n] = x[:n, :qh]
    ref.append(k, v, t["table"], t["starts"], t["lens"], x[:, qh:], t["qkv"][:, qh + kvh:])
    return q, k, v


def same(got, want):
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.view(np.uint16), b.view(np.uint16))


@pytest.mark.parametrize("layout", list(RopeLayout))
@pytest.mark.parametrize("new,past,qh,kvh,hd,pairs,block", [
    ([1], [0], 4, 1, 64, 32, 16), ([1] * 9, [0, 15, 16, 31, 5, 100, 47, 48, 1], 8, 2, 128, 64, 16),
    ([33, 0, 1, 70], [0, 9, 31, 2], 32, 8, 64, 32, 32), ([5, 300], [60, 0], 5, 5, 128, 32, 64),
    ([17], [250], 7, 1, 64, 8, 256), ([40, 41], [7, 0], 3, 1, 128, 5, 48),
    ([2, 3], [0, 0], 2, 2, 64, 0, 16), ([129], [0], 16, 1, 128, 64, 128),
    ([100], [3], 1, 4, 64, 1, 96), ([20, 9], [0, 4], 12, 3, 128, 12, 80)])
def test_rows_land_rotated(ctx, layout, new, past, qh, kvh, hd, pairs, block):
    t = inputs(new, past, qh, kvh, hd, pairs, block, seed=len(new) + hd)
    same(run(ctx, t, layout), expected(t, layout))


def test_within_half_a_step_of_64_bits(ctx):
    """Half a step of the f16 result, half a step of each of three f32 operations."""
    t = inputs([50], [0], 4, 2, 128, 64, 32, seed=5)
    q, _, _ = run(ctx, t)
    x, c, s = t["qkv"][:, :4].astype(np.float64), t["cos"][:, None].astype(np.float64), t["sin"][:, None].astype(np.float64)
    a, b = x[..., :64], x[..., 64:]
    want = np.concatenate([a * c - b * s, b * c + a * s], -1)
    room = np.concatenate([abs(a * c) + abs(b * s)] * 2, -1)
    assert (np.abs(q - want) <= np.abs(want) * 2.0 ** -11 + room * 2.0 ** -22 + 2.0 ** -25).all()


def test_q_equals_the_rope_operator(ctx):
    t = inputs([33, 20], [0, 50], 8, 2, 128, 32, 16, seed=6)
    q, _, _ = run(ctx, t)
    src, out = put(ctx, t["qkv"][:, :8]), ctx.empty(plain((53, 8, 128), DType.F16))
    ops.rope_f16(ctx, src, put(ctx, t["cos"]), put(ctx, t["sin"]), out, 64, RopeLayout.HalfSplit)
    np.testing.assert_array_equal(q.view(np.uint16), get(ctx, out).view(np.uint16))


def test_not_finite_values_stay_where_they_are(ctx):
    """Infinities and NaN reach their own pair and no other; v is copied as it is."""
    t = inputs([21], [3], 4, 2, 64, 16, 16, seed=7)
    t["qkv"][3, 1, 5] = np.inf
    t["qkv"][4, 4, 60] = np.nan
    t["qkv"][5, 7, :] = -np.inf
    with np.errstate(invalid="ignore"):
        want = expected(t)
    for a, b in zip(run(ctx, t), want):
        np.testing.assert_array_equal(np.isnan(a), np.isnan(b))
        np.testing.assert_array_equal(np.nan_to_num(a), np.nan_to_num(b))


def test_rows_behind_the_last_sequence_are_left(ctx):
    t = inputs([3, 0, 18], [0, 0, 40], 4, 2, 64, 32, 16, seed=8, tail=11)
    same(run(ctx, t), expected(t))


def test_rows_before_the_first_sequence_are_left(ctx):
    t = inputs([3, 18], [0, 40], 4, 2, 64, 32, 16, seed=13)
    want = expected(t)
    q0, t["q_out"] = t["q_out"], np.concatenate([t["q_out"][:4], t["q_out"]])
    for n in ("qkv", "cos", "sin"):
        t[n] = np.concatenate([t[n][:4], t[n]])
    t["starts"] = t["starts"] + 4
    q, k, v = run(ctx, t)
    same((q[:4], q[4:], k, v), (q0[:4], *want))


@pytest.mark.parametrize("batch", [33, 700])
def test_many_sequences(ctx, batch):
    t = inputs([i % 4 for i in range(batch)], [(7 * i) % 50 for i in range(batch)], 4, 2, 64, 32, 16, seed=batch)
    same(run(ctx, t), expected(t))


def test_empty_sequences_everywhere(ctx):
    t = inputs([0, 0, 4, 0, 0, 1, 0], [0, 9, 0, 3, 0, 20, 1], 4, 2, 64, 32, 16, seed=9)
    same(run(ctx, t), expected(t))


@pytest.mark.parametrize("what", ["length below the rows", "length past the table", "starts fall",
                                  "starts past the rows", "block", "block below", "starts below"])
def test_out_of_range(ctx, what):
    """What is out of range is skipped, the rest written, and the call raises."""
    t = inputs([5, 6, 7], [20, 0, 3], 4, 2, 64, 32, 16, seed=10)
    good = {n: a.copy() for n, a in t.items()}
    skipped = 1
    if what == "length below the rows":
        t["lens"][1] = 5
    elif what == "length past the table":
        t["lens"][1] = 16 * t["table"].shape[1] + 1
    elif what == "starts fall":
        t["starts"][1], t["starts"][2] = 11, 5
        skipped = None
    elif what == "starts below":
        t["starts"][0] = -1
        skipped = 0
    elif what == "starts past the rows":
        t["starts"][3] = 19
        skipped = 2
    else:
        t["table"][1, 0] = len(t["k_cache"]) if what == "block" else -5
    held = {n: put(ctx, a) for n, a in t.items()}
    with pytest.raises(errors.IndexOutOfRange):
        ops.rope_kv_cache_append_paged_f16(ctx, *held.values())
    got = tuple(get(ctx, held[n]) for n in ("q_out", "k_cache", "v_cache"))
    if skipped is None:
        return  # which rows are whose is not defined; nothing faulted
    want = expected(good)
    rows = slice(good["starts"][skipped], good["starts"][skipped + 1])
    if not what.startswith("block"):
        want[0][rows] = t["q_out"][rows]
    for b in [skipped]:
        blocks = good["table"][b][good["table"][b] >= 0]
        want[1][blocks], want[2][blocks] = t["k_cache"][blocks], t["v_cache"][blocks]
    same(got, want)
    ops.rope_kv_cache_append_paged_f16(ctx, *held.values(), check=False)
    assert ctx.device_status() & 2


def test_replays_from_a_graph(ctx):
    """A captured step that is replayed with the lengths advanced between."""
    import torch

    t = inputs([1] * 4, [0, 15, 30, 2], 4, 2, 64, 32, 16, seed=11)
    t["table"], blocks = ref.tables_of([3, 18, 33, 5], 16, np.random.default_rng(1))
    t["k_cache"] = t["v_cache"] = np.zeros((blocks, 2, 16, 64), np.float16)
    held = {n: put(ctx, a) for n, a in t.items()}
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(ctx.stream)
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        ops.rope_kv_cache_append_paged_f16(ctx, *held.values(), check=False)
    want = None
    for _ in range(3):
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.sync()
        want = expected(t if want is None else t | {"k_cache": want[1], "v_cache": want[2]})
        t["lens"] = t["lens"] + 1
        ctx.upload_numpy(held["lens"], t["lens"])
    same(tuple(get(ctx, held[n]) for n in ("q_out", "k_cache", "v_cache")), want)


def test_without_tables(ctx):
    """No pairs: rows are copied; the C entry takes null tables."""
    t = inputs([9], [4], 4, 2, 64, 0, 16, seed=12)
    held = {n: put(ctx, a) for n, a in t.items()}
    args = [h.pointer if n not in ("cos", "sin") else None for n, h in held.items()]
    assert lib().mote_cuda_rope_kv_cache_append_paged_f16(
        *args, 9, 1, 4, 2, 64, 0, t["k_cache"].shape[0], 16, t["table"].shape[1], 0, None, ctx.stream) == 0
    same(tuple(get(ctx, held[n]) for n in ("q_out", "k_cache", "v_cache")), expected(t))
