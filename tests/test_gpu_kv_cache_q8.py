"""GPU parity of the KV cache held in 8 bits: append, read back and decode
attention, and a serving run of them with the packed prompt attention.

Append and read are compared bit for bit with the definition
(tests/_q8_cache.py); attention with the definition in 64 bits over the
cache's own values, at the bound derived in ``check_attention``.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200 import errors, ops  # noqa: E402
from mote_b200.context import CudaContext  # noqa: E402
from mote_b200.types import DType, plain  # noqa: E402
from tests import _q8_cache as ref  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


def up(ctx, a, dtype):
    return ctx.from_bytes(plain(a.shape, dtype), a)


def i32(ctx, a):
    a = np.ascontiguousarray(a, dtype=np.int32)
    return up(ctx, a, DType.I32)


def f16(ctx, a):
    return up(ctx, np.ascontiguousarray(a, dtype=np.float16), DType.F16)


def starts_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


class Cache:
    """A cache on the device beside its host definition, pages in no order."""

    def __init__(self, ctx, need, kvh, hd, bt, seed, spare=2):
        r = np.random.default_rng(seed)
        need = [-(-n // bt) for n in need]
        blocks = sum(need) + spare
        order = r.permutation(blocks).astype(np.int32)
        self.table = np.full((len(need), max(max(need), 1)), -1, np.int32)
        at = starts_of(need)
        for b, n in enumerate(need):
            self.table[b, :n] = order[at[b]:at[b + 1]]
        self.ctx, self.bt = ctx, bt
        # what was never written holds anything, NaN scales among it
        self.host = {n: r.integers(-128, 128, (blocks, kvh, bt, hd)).astype(np.int8) for n in "kv"}
        self.scale = {n: np.where(r.random((blocks, kvh)) < 0.5, np.nan, 3.0).astype(np.float32)
                      for n in "kv"}
        self.dev = {n: up(ctx, self.host[n], DType.I8) for n in "kv"}
        self.dscale = {n: up(ctx, self.scale[n], DType.F32) for n in "kv"}
        self.dtable = i32(ctx, self.table)

    @property
    def tensors(self):
        return (self.dev["k"], self.dev["v"], self.dscale["k"], self.dscale["v"], self.dtable)

    def append(self, k, v, lens_after, starts, on_host=True, **kw):
        ops.kv_cache_append_q8(self.ctx, f16(self.ctx, k), f16(self.ctx, v), *self.tensors,
                               i32(self.ctx, starts), i32(self.ctx, lens_after), **kw)
        if on_host:
            for n, x in (("k", k), ("v", v)):
                ref.append(self.host[n], self.scale[n], self.table, x, lens_after, starts)

    def check(self):
        for n in "kv":
            got = np.frombuffer(self.ctx.read_bytes(self.dev[n]), np.int8).reshape(self.host[n].shape)
            assert np.array_equal(got, self.host[n]), n
            got = np.frombuffer(self.ctx.read_bytes(self.dscale[n]), np.float32)
            assert np.array_equal(got, self.scale[n].ravel(), equal_nan=True), n

    def decode(self, q, lens, scale=None):
        out = f16(self.ctx, np.full(q.shape, np.nan))
        ops.gqa_attention_decode_q8(self.ctx, f16(self.ctx, q), *self.tensors, i32(self.ctx, lens),
                                    out, scale)
        return np.frombuffer(self.ctx.read_bytes(out), np.float16).reshape(q.shape)

    def check_decode(self, q, lens, scale=None):
        got = self.decode(q, lens, scale)
        for b, n in enumerate(lens):
            if n == 0:
                assert (got[b] == 0).all()
                continue
            k, v = (ref.rows(self.host[m], self.scale[m], self.table[b], n) for m in "kv")
            ref.check_attention(got[b:b + 1], *ref.attention(
                q[b:b + 1], k, v, [n], ref.default_scale(q.shape[2]) if scale is None else scale))
        return got


def keys(r, n, kvh, hd, gain=1.0):
    """f16 rows with channels that stand out."""
    x = r.normal(0, gain, (n, kvh, hd))
    x[:, :, 3::37] *= 6
    return x.astype(np.float16)


@pytest.mark.parametrize("kvh,hd,bt,past,new", [
    (1, 64, 16, [0], [1]), (2, 128, 16, [0, 0], [33, 0]), (3, 64, 32, [5, 31, 32], [1, 2, 70]),
    (8, 128, 64, [0, 1, 63, 64, 100], [200, 64, 1, 63, 29]), (2, 64, 256, [255, 3], [2, 300]),
    (8, 64, 48, [0, 47, 96], [0, 1, 49]), (1, 128, 128, [0] * 40, list(range(40)))])
def test_append_is_the_definition_bit_for_bit(ctx, kvh, hd, bt, past, new):
    r = np.random.default_rng(kvh * 1000 + bt)
    past, new = np.array(past), np.array(new)
    c = Cache(ctx, past + new, kvh, hd, bt, seed=bt)
    for lens, n in ((past, past), (past + new, new)):
        total = int(n.sum())
        # the second call's rows are larger in some heads, smaller in others
        gain = np.where(np.arange(kvh) % 2, 0.3, 4.0)[None, :, None]
        k, v = keys(r, total, kvh, hd) * gain, keys(r, total, kvh, hd) / gain
        c.append(k.astype(np.float16), v.astype(np.float16), lens, starts_of(n))
        c.check()
    assert ctx.device_status() == 0


def test_append_one_by_one_with_growing_rows(ctx):
    """Single tokens whose size grows and shrinks: the block is rounded again
    each time its scale grows, exact ties (half the largest) among them."""
    kvh, hd, bt = 2, 64, 16
    r = np.random.default_rng(8)
    c = Cache(ctx, [40, 40], kvh, hd, bt, seed=3)
    for i in range(40):
        k = keys(r, 2, kvh, hd, gain=2.0 ** r.integers(-6, 7))
        k[0, 0, :8] = np.abs(k[0, 0]).max() * np.array([1, .5, -.5, .25, -1, 0, .5, .75])
        c.append(k, keys(r, 2, kvh, hd), [i + 1, i + 1], [0, 1, 2])
    c.check()
    c.check_decode(r.normal(0, 1, (2, 8, hd)).astype(np.float16), [40, 40])


def test_append_extremes_and_values_that_are_not_finite(ctx):
    kvh, hd, bt = 2, 64, 16
    c = Cache(ctx, [32], kvh, hd, bt, seed=4)
    z = np.zeros((3, kvh, hd), np.float16)
    c.append(z, z, [3], [0, 3])  # all zeros: scale 0
    c.check()
    tiny = np.full((1, kvh, hd), 6e-8, np.float16)  # the smallest f16
    c.append(tiny, -tiny, [4], [0, 1])
    huge = np.full((1, kvh, hd), 65504, np.float16)
    c.append(huge, -huge, [5], [0, 1])
    c.check()
    bad = np.ones((1, kvh, hd), np.float16)
    bad[0, 0, 5] = np.inf  # head 0 of K reads as NaN from here on, head 1 does not
    c.append(bad, np.ones_like(bad), [6], [0, 1])
    c.append(np.ones_like(bad), np.ones_like(bad), [7], [0, 1])
    c.check()
    assert np.isnan(c.scale["k"][c.table[0, 0], 0]) and np.isfinite(c.scale["k"][c.table[0, 0], 1])
    bad[0, 0, 5] = np.nan
    c.append(np.ones_like(bad), bad, [17], [0, 1])
    c.check()
    got = c.decode(np.ones((1, kvh, hd), np.float16), [7])
    assert np.isnan(got[0, 0]).all() and np.isfinite(got[0, 1]).all()
    c.append(np.ones_like(bad), np.ones_like(bad), [1], [0, 1])  # its first row again
    c.check()
    assert np.isfinite(c.scale["k"][c.table[0, 0]]).all()


def test_append_refuses_bad_offsets_lengths_and_blocks(ctx):
    kvh, hd, bt = 2, 64, 16
    r = np.random.default_rng(5)
    c = Cache(ctx, [32, 32, 32], kvh, hd, bt, seed=5)
    k, v = keys(r, 9, kvh, hd), keys(r, 9, kvh, hd)

    def host(b, lo, hi, length):
        for n, x in (("k", k), ("v", v)):
            ref.append(c.host[n], c.scale[n], c.table[b:b + 1], x[lo:hi], [length], [0, hi - lo])

    for starts, lens, good in (
            ([0, 3, 6, 10], [3, 3, 4], [(0, 0, 3, 3), (1, 3, 6, 3)]),    # past the last row
            ([0, 3, 6, 9], [3, 2, 3], [(0, 0, 3, 3), (2, 6, 9, 3)]),     # shorter than its rows
            ([0, 3, 6, 9], [3, 34, 3], [(0, 0, 3, 3), (2, 6, 9, 3)]),    # past the table's blocks
            ([-1, 3, 6, 9], [4, 3, 3], [(1, 3, 6, 3), (2, 6, 9, 3)])):
        with pytest.raises(errors.IndexOutOfRange):
            c.append(k, v, lens, starts, on_host=False)
        for g in good:
            host(*g)
        if lens[1] == 34:  # the row that the sequence's second block still takes
            host(1, 3, 4, 32)
        c.check()
    assert ctx.device_status() == 0  # told by the exception alone
    table = c.table.copy()
    for block in (-1, c.host["k"].shape[0], -2**31, 2**31 - 1):
        c.table[1, 0] = block
        c.dtable = i32(ctx, c.table)
        c.append(k, v, [3, 3, 3], [0, 3, 6, 9], on_host=False, check=False)
        assert ctx.device_status() == 2
        assert ctx.device_status() == 0
        host(0, 0, 3, 3), host(2, 6, 9, 3)
        c.check()
        out = [f16(ctx, np.full((9, kvh, hd), 7.0)) for _ in "kv"]
        with pytest.raises(errors.IndexOutOfRange):
            ops.kv_cache_read_q8(ctx, *c.tensors, i32(ctx, [0, 3, 6, 9]), *out)
        got = np.frombuffer(ctx.read_bytes(out[0]), np.float16).reshape(9, kvh, hd)
        assert (got[3:6] == 7).all()
    c.table[:] = table


@pytest.mark.parametrize("kvh,hd,bt,lens", [(1, 64, 16, [1]), (8, 128, 64, [0, 130, 1, 64]),
                                            (2, 128, 256, [300, 5]), (3, 64, 48, [47, 0, 0, 100])])
def test_read_gives_the_values_and_leaves_other_rows(ctx, kvh, hd, bt, lens):
    r = np.random.default_rng(11)
    c = Cache(ctx, lens, kvh, hd, bt, seed=6)
    total = sum(lens)
    c.append(keys(r, total, kvh, hd), keys(r, total, kvh, hd), lens, starts_of(lens))
    before, behind = 2, 3  # rows of no sequence at both ends
    out = [f16(ctx, np.full((before + total + behind, kvh, hd), 7.0)) for _ in "kv"]
    ops.kv_cache_read_q8(ctx, *c.tensors, i32(ctx, starts_of(lens) + before), *out)
    for n, t in zip("kv", out):
        got = np.frombuffer(ctx.read_bytes(t), np.float16).reshape(-1, kvh, hd)
        want = np.concatenate([ref.rows(c.host[n], c.scale[n], c.table[b], m)
                               for b, m in enumerate(lens)]).astype(np.float16)
        assert np.array_equal(got[before:before + total], want)
        assert (got[:before] == 7).all() and (got[before + total:] == 7).all()
    assert ctx.device_status() == 0


@pytest.mark.parametrize("qh,kvh,hd,bt,lens", [
    (32, 8, 64, 16, [1]), (32, 8, 128, 16, [117]), (32, 8, 64, 32, [0, 1, 15, 16, 17, 31, 33]),
    (32, 8, 128, 64, [300, 0, 64, 63, 65, 1]), (1, 1, 64, 128, [129]), (8, 8, 128, 16, [40, 2]),
    (5, 1, 64, 48, [500]), (21, 3, 128, 64, [200, 7]), (16, 1, 128, 256, [700]),
    (24, 2, 64, 16, [90, 300]), (40, 2, 128, 32, [77]), (6, 2, 64, 64, [1000, 3, 0])])
def test_decode_matches_the_definition(ctx, qh, kvh, hd, bt, lens):
    r = np.random.default_rng(qh * 100 + hd)
    c = Cache(ctx, lens, kvh, hd, bt, seed=qh)
    total = sum(lens)
    c.append(keys(r, total, kvh, hd), r.normal(0, 1, (total, kvh, hd)).astype(np.float16), lens,
             starts_of(lens))
    q = r.normal(0, 1, (len(lens), qh, hd)).astype(np.float16)
    c.check_decode(q, lens)
    c.check_decode(q, [n // 2 for n in lens], scale=0.3)  # shorter than what is cached
    c.check_decode(q, lens, scale=-0.05)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("hd,batch,length", [(64, 1, 5000), (128, 1, 9000), (128, 3, 2500),
                                             (64, 40, 300)])
def test_decode_split_over_positions(ctx, hd, batch, length):
    """Long rows whose parts are joined; values of one size, so that the
    output's rounding shows."""
    r = np.random.default_rng(hd + length)
    lens = [max(1, length - 37 * b) for b in range(batch)]
    c = Cache(ctx, lens, 4, hd, 64, seed=batch)
    total = sum(lens)
    v = 2.0 + 0.1 * r.normal(0, 1, (total, 4, hd))
    c.append(keys(r, total, 4, hd), v.astype(np.float16), lens, starts_of(lens))
    q = r.normal(0, 1, (batch, 16, hd)).astype(np.float16)
    a = c.check_decode(q, lens)
    assert np.array_equal(a, c.decode(q, lens))  # the same again
    assert ctx.device_status() == 0


def test_decode_rows_that_dominate_and_vanish(ctx):
    """A first position far above the rest, whose V is small (an attention
    sink), and scores that grow along the row (the running maximum moves)."""
    r = np.random.default_rng(21)
    n, kvh, hd = 1200, 2, 128
    k = r.normal(0, 0.1, (n, kvh, hd))
    q = np.ones((2, 8, hd))
    k[0, 0] += 12.0 / np.sqrt(hd)           # head 0: +12 over the others
    k[:, 1] += np.linspace(0, 40, n)[:, None] / np.sqrt(hd) / 4  # head 1: grows by 10
    v = r.normal(0, 1, (n, kvh, hd))
    v[:64] *= 2.0 ** -10                     # the first block's scale is small too
    c = Cache(ctx, [n, n], kvh, hd, 64, seed=22)
    c.append(np.concatenate([k, k[::-1]]).astype(np.float16),
             np.concatenate([v, v[::-1]]).astype(np.float16), [n, n], [0, n, 2 * n])
    c.check_decode(q.astype(np.float16), [n, n])


def test_decode_blocks_out_of_range_count_as_not_there(ctx):
    r = np.random.default_rng(31)
    kvh, hd, bt, n = 2, 128, 16, 100
    c = Cache(ctx, [n], kvh, hd, bt, seed=31)
    k, v = keys(r, n, kvh, hd), keys(r, n, kvh, hd)
    c.append(k, v, [n], [0, n])
    q = r.normal(0, 1, (1, 8, hd)).astype(np.float16)
    kv = [ref.rows(c.host[m], c.scale[m], c.table[0], n) for m in "kv"]
    gone = np.zeros(n, bool)
    for i, block in ((0, -1), (3, 1 << 30), (6, -2**31)):
        c.table[0, i] = block
        gone[i * bt:(i + 1) * bt] = True
    c.dtable = i32(ctx, c.table)
    got = c.decode(q, [n])
    assert ctx.device_status() == 2
    ref.check_attention(got, *ref.attention(q, kv[0][~gone], kv[1][~gone], [n],
                                            ref.default_scale(hd)))
    # lengths past the table and below zero
    c.table[0] = np.arange(c.table.shape[1])
    c.dtable = i32(ctx, c.table)
    c.scale = {m: np.ones_like(s) for m, s in c.scale.items()}
    c.dscale = {m: up(ctx, s, DType.F32) for m, s in c.scale.items()}
    whole = c.check_decode(q, [c.table.shape[1] * bt], scale=0.001)
    assert np.array_equal(c.decode(q, [2**31 - 1], scale=0.001), whole)
    assert (c.decode(q, [-5]) == 0).all()
    assert ctx.device_status() == 0


def test_offsets_past_32_bits(ctx):
    """Blocks whose bytes begin past 2^32: 5 GB of K and V each."""
    kvh, hd, bt, n = 8, 128, 256, 700
    blocks = (5 << 30) // (kvh * bt * hd)
    r = np.random.default_rng(41)
    k, v = keys(r, n, kvh, hd), keys(r, n, kvh, hd)
    dev = [ctx.empty(plain((blocks, kvh, bt, hd), DType.I8)) for _ in "kv"]
    scales = [ctx.empty(plain((blocks, kvh), DType.F32)) for _ in "kv"]
    table = np.array([[blocks - 1, blocks - 9, blocks - 4]], np.int32)
    args = (*dev, *scales, i32(ctx, table))
    ops.kv_cache_append_q8(ctx, f16(ctx, k), f16(ctx, v), *args, i32(ctx, [0, n]), i32(ctx, [n]))
    small = Cache(ctx, [n], kvh, hd, bt, seed=42)
    small.append(k, v, [n], [0, n])
    out = [f16(ctx, np.zeros((n, kvh, hd))) for _ in "kv"]
    ops.kv_cache_read_q8(ctx, *args, i32(ctx, [0, n]), *out)
    for m, t in zip("kv", out):
        want = ref.rows(small.host[m], small.scale[m], small.table[0], n).astype(np.float16)
        assert np.array_equal(np.frombuffer(ctx.read_bytes(t), np.float16), want.ravel())
    q = r.normal(0, 1, (1, 32, hd)).astype(np.float16)
    o = f16(ctx, np.zeros(q.shape))
    ops.gqa_attention_decode_q8(ctx, f16(ctx, q), *args, i32(ctx, [n]), o)
    got = np.frombuffer(ctx.read_bytes(o), np.float16).reshape(q.shape)
    assert np.array_equal(got, small.check_decode(q, [n]))


def test_a_serving_run_prompt_then_tokens_in_a_graph(ctx):
    """Packed prompts -> append -> decode steps replayed from one captured
    graph -> the cache read back under a continued prompt."""
    import torch

    qh, kvh, hd, bt, steps = 8, 2, 64, 16, 21
    r = np.random.default_rng(51)
    lens = np.array([37, 1, 64])
    c = Cache(ctx, lens + steps, kvh, hd, bt, seed=52)
    starts, total = starts_of(lens), int(lens.sum())
    q = r.normal(0, 1, (total, qh, hd)).astype(np.float16)
    k, v = keys(r, total, kvh, hd), keys(r, total, kvh, hd)
    out = f16(ctx, np.full(q.shape, np.nan))
    dk, dv, ds = f16(ctx, k), f16(ctx, v), i32(ctx, starts)
    ops.gqa_attention_packed_f16(ctx, f16(ctx, q), dk, dv, ds, ds, out)
    c.append(k, v, lens, starts)
    got = np.frombuffer(ctx.read_bytes(out), np.float16).reshape(q.shape)
    for b in range(3):
        s = slice(starts[b], starts[b + 1])
        ref.check_attention(got[s], *ref.attention(q[s], k[s], v[s], np.arange(1, lens[b] + 1),
                                                   ref.default_scale(hd)))
    one = i32(ctx, [0, 1, 2, 3])
    tk, tv, tq = (f16(ctx, np.zeros((3, h, hd))) for h in (kvh, kvh, qh))
    to, tl = f16(ctx, np.zeros((3, qh, hd))), i32(ctx, lens)

    def step():
        ops.kv_cache_append_q8(ctx, tk, tv, *c.tensors, one, tl, check=False)
        ops.gqa_attention_decode_q8(ctx, tq, *c.tensors, tl, to)

    graph = None
    for i in range(steps):
        n = lens + i + 1
        kn, vn = keys(r, 3, kvh, hd, 1.5), keys(r, 3, kvh, hd, 1.5)
        qn = r.normal(0, 1, (3, qh, hd)).astype(np.float16)
        for t, a in ((tk, kn), (tv, vn), (tq, qn), (tl, n.astype(np.int32))):
            ctx.upload_numpy(t, a)
        if i == 0:
            step()
        elif i == 1:
            graph = torch.cuda.CUDAGraph()
            stream = torch.cuda.ExternalStream(ctx.stream)
            with torch.cuda.graph(graph, stream=stream):
                step()
        if graph is not None:
            with torch.cuda.stream(stream):
                graph.replay()
        ctx.sync()
        for m, x in (("k", kn), ("v", vn)):
            ref.append(c.host[m], c.scale[m], c.table, x, n, [0, 1, 2, 3])
        got = np.frombuffer(ctx.read_bytes(to), np.float16).reshape(3, qh, hd)
        for b in range(3):
            kk, vv = (ref.rows(c.host[m], c.scale[m], c.table[b], int(n[b])) for m in "kv")
            ref.check_attention(got[b:b + 1], *ref.attention(qn[b:b + 1], kk, vv, [n[b]],
                                                             ref.default_scale(hd)))
    c.check()
    del graph
    # a continued prompt of 5 tokens each over everything cached
    n = lens + steps
    ks = starts_of(n)
    ko, vo = (f16(ctx, np.zeros((int(n.sum()), kvh, hd))) for _ in "kv")
    ops.kv_cache_read_q8(ctx, *c.tensors, i32(ctx, ks), ko, vo)
    q = r.normal(0, 1, (15, qh, hd)).astype(np.float16)
    out = f16(ctx, np.full(q.shape, np.nan))
    ops.gqa_attention_packed_f16(ctx, f16(ctx, q), ko, vo, i32(ctx, [0, 5, 10, 15]), i32(ctx, ks),
                                 out)
    got = np.frombuffer(ctx.read_bytes(out), np.float16).reshape(q.shape)
    for b in range(3):
        kk, vv = (ref.rows(c.host[m], c.scale[m], c.table[b], int(n[b])).astype(np.float16)
                  for m in "kv")
        ref.check_attention(got[5 * b:5 * b + 5], *ref.attention(
            q[5 * b:5 * b + 5], kk, vv, n[b] - 4 + np.arange(5), ref.default_scale(hd)))
    assert ctx.device_status() == 0


def test_two_contexts_at_once(ctx):
    """Each context has its own stream and workspace."""
    r = np.random.default_rng(61)
    lens = [3000, 10]
    caches = [Cache(x, lens, 8, 128, 64, seed=62) for x in (ctx, CudaContext(0))]
    k, v = keys(r, 3010, 8, 128), keys(r, 3010, 8, 128)
    q = r.normal(0, 1, (2, 32, 128)).astype(np.float16)
    for c in caches:
        c.append(k, v, lens, starts_of(lens))
    outs = [[f16(c.ctx, q) for _ in range(20)] for c in caches]
    ins = [(f16(c.ctx, q), i32(c.ctx, lens)) for c in caches]
    for i in range(20):
        for c, o, (tq, tl) in zip(caches, outs, ins):
            ops.gqa_attention_decode_q8(c.ctx, tq, *c.tensors, tl, o[i])
    want = caches[0].check_decode(q, lens)
    for c, o in zip(caches, outs):
        for t in o:
            assert np.array_equal(np.frombuffer(c.ctx.read_bytes(t), np.float16).reshape(q.shape),
                                  want)


@pytest.mark.parametrize("batch,kvh,top", [(16, 2, 300), (17, 2, 300), (1000, 1, 40), (400, 2, 90)])
def test_decode_finds_its_share_of_any_batch(ctx, batch, kvh, top):
    """Ragged batches around the sizes where the work is dealt another way,
    empty sequences among them, and one that is much longer."""
    r = np.random.default_rng(batch)
    lens = r.integers(0, top, batch)
    lens[r.integers(0, batch, batch // 5)] = 0
    lens[batch // 2] = 1500
    c = Cache(ctx, lens, kvh, 64, 32, seed=batch)
    total = int(lens.sum())
    c.append(keys(r, total, kvh, 64), keys(r, total, kvh, 64), lens, starts_of(lens))
    c.check()
    c.check_decode(r.normal(0, 1, (batch, 4 * kvh, 64)).astype(np.float16), lens)
    assert ctx.device_status() == 0


def test_graphs_that_share_the_workspace_take_turns(ctx):
    """Two captured graphs of different shapes and an eager call use one
    workspace one after another, in any order."""
    import torch

    r = np.random.default_rng(71)
    runs = []
    for hd, lens in ((128, [4000, 100]), (64, [900] * 30), (128, [20000])):
        c = Cache(ctx, lens, 2, hd, 64, seed=hd + len(lens))
        total = sum(lens)
        c.append(keys(r, total, 2, hd), keys(r, total, 2, hd), lens, starts_of(lens))
        q = r.normal(0, 1, (len(lens), 8, hd)).astype(np.float16)
        runs.append((c, f16(ctx, q), i32(ctx, lens), f16(ctx, np.zeros_like(q)),
                     c.check_decode(q, lens)))
    stream = torch.cuda.ExternalStream(ctx.stream)

    def call(run):
        c, q, lens, out, _ = run
        ops.gqa_attention_decode_q8(ctx, q, *c.tensors, lens, out)

    graphs = []
    for run in runs[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            call(run)
    for order in ([0, 1, 2], [2, 1, 0], [1, 1, 0, 0, 2]):
        for t in runs:
            ctx.upload_numpy(t[3], np.full(t[4].shape, np.nan, np.float16))
        for i in order:
            if i < 2:
                with torch.cuda.stream(stream):
                    graphs[i].replay()
            else:
                call(runs[2])
        for run in runs:
            got = np.frombuffer(ctx.read_bytes(run[3]), np.float16).reshape(run[4].shape)
            assert np.array_equal(got, run[4])
    del graphs
    assert ctx.device_status() == 0


def test_workspace_and_registry(ctx):
    """The C entry refuses a missing, small or unaligned workspace; through
    the kernel registry it takes the same words."""
    import ctypes

    from mote_b200 import kernel
    from mote_b200._native import lib

    r = np.random.default_rng(81)
    c = Cache(ctx, [50, 700], 2, 128, 16, seed=81)
    c.append(keys(r, 750, 2, 128), keys(r, 750, 2, 128), [50, 700], [0, 50, 750])
    q = r.normal(0, 1, (2, 8, 128)).astype(np.float16)
    want = c.check_decode(q, [50, 700])
    need = ctypes.c_uint64(0)
    assert lib().mote_cuda_gqa_attention_decode_q8_workspace_bytes(2, 8, 2, 128,
                                                                   ctypes.byref(need)) == 0
    ws = ctx.from_bytes(plain((need.value + 16,), DType.U8), np.zeros(need.value + 16, np.uint8))
    tq, tl, to = f16(ctx, q), i32(ctx, [50, 700]), f16(ctx, np.zeros_like(q))
    ptrs = [t.pointer for t in (tq, *c.tensors, tl, to)]
    blocks, kvh, bt, hd = c.host["k"].shape
    shape = (2, 8, kvh, hd, blocks, bt, c.table.shape[1])
    scale = ref.default_scale(hd)
    for pointer, size in ((None, 0), (ws.pointer, need.value - 1), (ws.pointer + 8, need.value)):
        assert lib().mote_cuda_gqa_attention_decode_q8(*ptrs, *shape, scale, pointer, size,
                                                       ctx.stream) == 1
    runtime = kernel.Runtime()
    kernel.register_cuda_kernels(runtime.kernels_mut())
    k = runtime.resolve(kernel.KernelKey("gqa_attention_decode_q8", DType.F16), ctx.device)
    k.launch(ctx.device, kernel.KernelArgs((*ptrs, *shape, kernel.f32_bits(scale), ws.pointer,
                                            need.value, ctx.stream)))
    got = np.frombuffer(ctx.read_bytes(to), np.float16).reshape(q.shape)
    assert np.array_equal(got, want)
