"""Measured cases of the 8-bit KV cache and of attention over packed prompts.

Four operators that a serving program calls one after another:

* ``packed``: causal grouped-query attention over whole prompts of different
  lengths, packed back to back (f16);
* ``append``: new K/V rows into a paged cache held in 8 bits, with one f32
  scale per block of tokens and head;
* ``read``: the cached rows of every sequence back in f16, packed (what a
  prompt continued over cached blocks attends to);
* ``decode``: one query token per sequence over that cache.

Head layouts are 32 query / 8 KV heads with head_dim 64 and 128 (this
repository's decoder layers) and the extremes of the grouping.
"""
import math

import numpy as np
import torch

own = False

GARBAGE_SCALE = 7.0  # what a block that was never written may hold


# ------------------------------------------------------------------- cases --
def _packed(name, lens, batch, lo, hi, past=0, q_heads=32, kv_heads=8, head_dim=128):
    return {"name": name, "op": "packed", "lens": lens, "batch": batch, "lo": lo, "hi": hi,
            "past": past, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim}


def _cache(name, op, lens, batch, lo, hi, past=0, q_heads=32, kv_heads=8, head_dim=128, block=64):
    return {"name": name, "op": op, "lens": lens, "batch": batch, "lo": lo, "hi": hi, "past": past,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block}


def listed():
    return [
        # one short question: latency of a single small call
        _packed("packed_one_short", 1, 1, 23, 23, head_dim=64),
        # an ordinary batch of chat prompts of ragged lengths, 1B-sized heads
        _packed("packed_batch_d64", 2, 12, 60, 1000, head_dim=64),
        # chunks of long prompts continued over what is cached already
        _packed("packed_chunks_d128", 3, 6, 300, 1024, past=2500),
        # one long document at 8B-sized heads: the largest prompt
        _packed("packed_long_d128", 4, 1, 8192, 8192),
        # one new token for each of 32 running sequences (and the rows so far, read back)
        _cache("append_step", "append", 5, 32, 1, 1, past=100, block=16),
        # whole prompts of a batch written at once
        _cache("append_prompts", "append", 6, 16, 40, 2048, past=90),
        # a few hundred cached rows before a short continued prompt
        _cache("read_few_d64", "read", 7, 4, 30, 200, head_dim=64, block=32),
        # long cached prefixes before continued prompts
        _cache("read_long", "read", 8, 8, 1000, 6000),
        # one user, short context: latency
        _cache("decode_one_short", "decode", 9, 1, 117, 117, block=16),
        # one user, long context: the split over positions and its join
        _cache("decode_one_long", "decode", 10, 1, 32768, 32768),
        # a full batch at equal lengths, 1B-sized heads
        _cache("decode_batch_d64", "decode", 11, 16, 4096, 4096, head_dim=64),
        # a serving batch whose lengths differ by orders of magnitude
        _cache("decode_batch_ragged", "decode", 12, 48, 1, 8192),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _with_lo(rng, case):
    """The shortest length: sequences of a batch may be empty."""
    return case | {"lo": rng.randint(0 if case["batch"] > 1 else 1, case["hi"])}


def draw(rng):
    op = rng.choice(["packed", "append", "read", "decode"])
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16] if kv_heads < 8 else [1, 2, 4])
    c = {"op": op, "lens": rng.randrange(1, 1 << 30), "q_heads": kv_heads * group,
         "kv_heads": kv_heads, "head_dim": head_dim}
    if op == "packed":
        most = 32 * 8192 * 8192 // c["q_heads"]  # the largest listed case's scores of a head
        hi = min(_log_int(rng, 1, 8192), math.isqrt(most))
        past = min(rng.choice([0, 0, _log_int(rng, 1, 4096)]), (most // hi - hi) // 2)
        c |= {"batch": _log_int(rng, 1, min(64, most // (hi * (hi + 2 * past)))),
              "hi": hi, "past": past}
        return _with_lo(rng, c)
    c["block"] = rng.choice([16, 32, 64, 128])
    if op == "append":
        hi = _log_int(rng, 1, 2048)
        c |= {"batch": _log_int(rng, 1, min(64, 15000 // hi)), "hi": hi,
              "past": rng.choice([0, _log_int(rng, 1, 200)])}
    elif op == "read":
        hi = _log_int(rng, 1, 6000)
        c |= {"batch": _log_int(rng, 1, min(32, 28000 // hi)), "hi": hi, "past": 0}
    else:
        hi = _log_int(rng, 1, 32768)
        batch = _log_int(rng, 1, max(1, min(128, 190000 // hi)))
        c |= {"batch": batch, "hi": hi, "past": 0}
    return _with_lo(rng, c)


def _lengths(case):
    """(past, new) lengths of the sequences: [batch] each."""
    r = np.random.RandomState(case["lens"])
    new = r.randint(case["lo"], case["hi"] + 1, case["batch"]).astype(np.int64)
    if case["batch"] > 1:
        new[r.randint(case["batch"])] = case["hi"]
    past = r.randint(0, case["past"] + 1, case["batch"]).astype(np.int64)
    return past, new


def _starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def work(case):
    past, new = _lengths(case)
    qh, kvh, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    total = past + new
    if case["op"] == "packed":
        # query i of a sequence attends past + i + 1 positions
        pairs = int((new * past + new * (new + 1) // 2).sum())
        return {"bytes": 2 * hd * (2 * qh * int(new.sum()) + 2 * kvh * int(total.sum())),
                "flops": 4 * hd * qh * pairs}
    values = 2 * kvh * hd  # K and V values of one position
    blocks = int((-(-total // case["block"])).sum())
    held = blocks * (4 + 2 * kvh * 4)  # table entries and scales
    if case["op"] == "decode":
        rows = int(total.sum())
        return {"bytes": rows * values + held + 4 * qh * hd * case["batch"],
                "flops": 4 * hd * qh * rows}
    if case["op"] == "read":
        rows = int(total.sum())
        return {"bytes": rows * values * 3 + held, "flops": rows * values}
    # append: new rows read in f16 and written in 8 bits, then every row read back in f16
    rows = int(new.sum())
    return {"bytes": rows * values * 3 + int(total.sum()) * values * 3 + 2 * held,
            "flops": 2 * rows * values + int(total.sum()) * values}


# ------------------------------------------------------------------ inputs --
def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)


def _gains(gen, kv_heads, head_dim):
    """Channel gains of K: a few channels stand out, as keys' do."""
    g = torch.ones(kv_heads, 1, head_dim, device="cuda", dtype=torch.float16)
    g[:, :, torch.randint(0, head_dim, (2,), generator=gen, device="cuda")] = 4.0
    return g


def _inputs(case, seed):
    """The case's tensors from the seed, on the GPU."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 11)
    past, new = _lengths(case)
    total = past + new
    qh, kvh, hd, batch = case["q_heads"], case["kv_heads"], case["head_dim"], case["batch"]

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()

    if case["op"] == "packed":
        return {"q": _randn(gen, int(new.sum()), qh, hd), "k": _randn(gen, int(total.sum()), kvh, hd),
                "v": _randn(gen, int(total.sum()), kvh, hd), "q_starts": ints(_starts(new)),
                "kv_starts": ints(_starts(total))}
    bt = case["block"]
    need = -(-total // bt)
    width = int(need.max())
    num_blocks = int(need.sum()) + 3
    # pages in no order, unused table entries -1
    order = np.random.RandomState((int(seed) * 31 + 5) % (1 << 31)).permutation(num_blocks)
    table = np.full((batch, width), -1, np.int32)
    at = _starts(need)
    for b in range(batch):
        table[b, :need[b]] = order[at[b]:at[b + 1]]
    t = {"block_tables": ints(table), "seq_lens": ints(total), "read_starts": ints(_starts(total))}
    for name in ("k", "v"):
        x = _randn(gen, num_blocks, kvh, bt, hd)
        x = x * _gains(gen, kvh, hd) if name == "k" else x
        if case["op"] == "append":
            # rows of the past are in their blocks, the rest holds anything
            held = torch.zeros(num_blocks, bt, dtype=torch.bool, device="cuda")
            pos = torch.arange(width * bt, device="cuda").view(1, width, bt)
            live = pos < ints(past).view(-1, 1, 1)
            ok = t["block_tables"] >= 0
            held[t["block_tables"][ok].long()] = live[ok]
        else:
            held = torch.ones(num_blocks, bt, dtype=torch.bool, device="cuda")
        amax = (x.abs().amax(-1).float() * held[:, None, :]).amax(-1)
        scale = amax / 127.0
        inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
        q = (x.double() * inv[..., None, None].double()).round().clamp(-127, 127).to(torch.int8)
        t[name + "_cache"] = q
        t[name + "_scales"] = torch.where(held.any(-1)[:, None], scale,
                                          torch.full_like(scale, GARBAGE_SCALE))
    if case["op"] == "decode":
        t["q"] = _randn(gen, batch, qh, hd)
    elif case["op"] == "append":
        t["seq_starts"] = ints(_starts(new))
        t["k_new"] = (_randn(gen, int(new.sum()), kvh, 1, hd) * _gains(gen, kvh, hd)).view(-1, kvh, hd)
        t["v_new"] = _randn(gen, int(new.sum()), kvh, hd)
    return t


class _Memory:
    """A framework tensor's device memory as torch sees it."""

    def __init__(self, tensor, shape, typestr):
        self.tensor = tensor  # keeps the storage
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "version": 3,
                                         "data": (tensor.pointer, False), "strides": None}


_context = None


def _framework_tensors(tensors):
    """The same values in the framework's storage: ({name: Tensor}, {name: torch view})."""
    global _context
    from mote_b200 import context, types

    if _context is None:
        _context = context.CudaContext(0)
    kinds = {torch.float16: (types.DType.F16, "<f2"), torch.float32: (types.DType.F32, "<f4"),
             torch.int32: (types.DType.I32, "<i4"), torch.int8: (types.DType.I8, "|i1")}
    held, seen = {}, {}
    for name, x in tensors.items():
        dtype, typestr = kinds[x.dtype]
        held[name] = _context.empty(types.plain(tuple(x.shape), dtype))
        seen[name] = torch.as_tensor(_Memory(held[name], x.shape, typestr), device="cuda")
        seen[name].copy_(x)
    torch.cuda.synchronize()
    return held, seen


def prepare(case, seed):
    t = _inputs(case, seed)
    past, new = _lengths(case)
    total = int((past + new).sum())
    kvh, hd = case["kv_heads"], case["head_dim"]
    # a serving program knows its lengths
    state = {"case": case, "in": t, "rows": total, "most": (int(new.max()), int((past + new).max()))}
    if own:
        if case["op"] in ("packed", "decode"):
            outs = {"out": torch.zeros_like(t["q"])}
        else:
            outs = {n: torch.zeros(total, kvh, hd, dtype=torch.float16, device="cuda")
                    for n in ("k_out", "v_out")}
        state["held"], state["seen"] = _framework_tensors(t | outs)
        state["in"] = None
        state["context"] = _context
    return state


# ------------------------------------------------------------- plain forms --
def _rows(starts, count):
    """(sequence, index in it) of each of `count` packed rows."""
    row = torch.arange(count, device=starts.device)
    seq = torch.searchsorted(starts[1:].contiguous(), row.int(), right=True)
    return seq, row - starts[seq]


def _softmax_weights(scores, allowed):
    """Softmax over the last axis where `allowed`; rows without any get zeros."""
    scores = scores.masked_fill_(~allowed, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
    e = scores.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    return e, torch.where(total > 0, total, torch.ones_like(total))


def _plain_packed(t, most):
    q, k, v, qs, ks = t["q"], t["k"], t["v"], t["q_starts"], t["kv_starts"]
    qh, kvh, hd = q.shape[1], k.shape[1], q.shape[2]
    nq, nk = qs[1:] - qs[:-1], ks[1:] - ks[:-1]
    seq, idx = _rows(qs, q.shape[0])
    kseq, kidx = _rows(ks, k.shape[0])
    batch, (mq, mk) = nq.numel(), most
    pq = torch.zeros(batch, mq, qh, hd, device=q.device)
    pk = torch.zeros(batch, mk, kvh, hd, device=q.device)
    pv = torch.zeros(batch, mk, kvh, hd, device=q.device)
    pq[seq, idx], pk[kseq, kidx], pv[kseq, kidx] = q.float(), k.float(), v.float()
    pq = pq.view(batch, mq, kvh, qh // kvh, hd).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(pq * (1.0 / math.sqrt(hd)), pk.permute(0, 2, 3, 1).unsqueeze(2))
    last = (nk - nq).view(-1, 1) + torch.arange(mq, device=q.device)
    allowed = torch.arange(mk, device=q.device) <= last.unsqueeze(-1)
    e, total = _softmax_weights(scores, allowed[:, None, None])
    out = torch.matmul(e, pv.permute(0, 2, 1, 3).unsqueeze(2)) / total
    return out.permute(0, 3, 1, 2, 4).reshape(batch, mq, qh, hd)[seq, idx].half()


def _plain_read(cache, scales, table, starts, count):
    """The cached rows of every sequence, packed, in f16."""
    bt = cache.shape[2]
    seq, pos = _rows(starts, count)
    block = table[seq, pos // bt].long()
    return (cache[block, :, pos % bt].float() * scales[block][..., None]).half()


def _plain_append(x, cache, scales, table, starts, lens):
    """The cache and the scales after the new rows `x` of every sequence."""
    bt = cache.shape[2]
    seq, idx = _rows(starts, x.shape[0])
    pos = (lens - (starts[1:] - starts[:-1]))[seq] + idx
    block, off = table[seq, pos // bt].long(), pos % bt
    blocks, kvh = scales.shape
    amax = torch.zeros(blocks, kvh, device=x.device).index_reduce_(
        0, block, x.float().abs().amax(-1), "amax")
    first = torch.full((blocks,), bt, device=x.device).index_reduce_(0, block, off, "amin")
    old = torch.where((first == 0)[:, None], torch.zeros_like(scales), scales)
    new = torch.where((first < bt)[:, None], torch.maximum(old, amax / 127.0), scales)
    inv = torch.where(new > 0, 1.0 / new, torch.zeros_like(new))
    # rows already there, on the grown scale; products in 64 bits, where they are exact
    ratio = old * inv
    grown = (first < bt)[:, None] & (new != old)
    again = (cache.double() * ratio.double()[..., None, None]).round().to(torch.int8)
    before = torch.arange(bt, device=x.device) < first[:, None]
    cache = torch.where(grown[:, :, None, None] & before[:, None, :, None], again, cache)
    cache[block, :, off] = (x.double() * inv[block].double()[..., None]).round().to(torch.int8)
    return cache, new


def _plain_decode(t):
    q, table, lens = t["q"], t["block_tables"].clamp(min=0).long(), t["seq_lens"]
    batch, qh, hd = q.shape
    kvh = t["k_cache"].shape[1]

    def padded(name):  # [batch, kv_heads, positions, head_dim]
        c = t[name + "_cache"][table].float() * t[name + "_scales"][table][..., None, None]
        return c.permute(0, 2, 1, 3, 4).reshape(batch, kvh, -1, hd)

    k = padded("k")
    scores = torch.matmul(q.view(batch, kvh, qh // kvh, hd).float() * (1.0 / math.sqrt(hd)),
                          k.transpose(-1, -2))
    allowed = torch.arange(k.shape[2], device=q.device) < lens[:, None]
    e, total = _softmax_weights(scores, allowed[:, None, None])
    return (torch.matmul(e, padded("v")) / total).view(batch, qh, hd).half()


def run(state):
    op = state["case"]["op"]
    if own:
        from mote_b200 import ops

        c, h, seen = state["context"], state["held"], state["seen"]
        if op == "packed":
            ops.gqa_attention_packed_f16(c, h["q"], h["k"], h["v"], h["q_starts"], h["kv_starts"],
                                         h["out"])
            return seen["out"]
        if op == "decode":
            ops.gqa_attention_decode_q8(c, h["q"], h["k_cache"], h["v_cache"], h["k_scales"],
                                        h["v_scales"], h["block_tables"], h["seq_lens"], h["out"])
            return seen["out"]
        if op == "append":
            ops.kv_cache_append_q8(c, h["k_new"], h["v_new"], h["k_cache"], h["v_cache"],
                                   h["k_scales"], h["v_scales"], h["block_tables"],
                                   h["seq_starts"], h["seq_lens"], check=False)
        # the cache's values: what is held in 8 bits stands for these
        ops.kv_cache_read_q8(c, h["k_cache"], h["v_cache"], h["k_scales"], h["v_scales"],
                             h["block_tables"], h["read_starts"], h["k_out"], h["v_out"],
                             check=False)
        return seen["k_out"], seen["v_out"]
    t = state["in"]
    if op == "packed":
        return _plain_packed(t, state["most"])
    if op == "decode":
        return _plain_decode(t)
    k, v, ks, vs = t["k_cache"], t["v_cache"], t["k_scales"], t["v_scales"]
    if op == "append":
        k, ks = _plain_append(t["k_new"], k, ks, t["block_tables"], t["seq_starts"], t["seq_lens"])
        v, vs = _plain_append(t["v_new"], v, vs, t["block_tables"], t["seq_starts"], t["seq_lens"])
    return (_plain_read(k, ks, t["block_tables"], t["read_starts"], state["rows"]),
            _plain_read(v, vs, t["block_tables"], t["read_starts"], state["rows"]))


# ---------------------------------------------- the definitions in 64 bits --
def _attend(q, k, v, reach):
    """softmax(q k^T / sqrt(d)) v in 64 bits; row i attends the first reach[i] positions."""
    s = (q @ k.T) / math.sqrt(q.shape[-1])
    s = s.masked_fill(torch.arange(k.shape[0], device=q.device) >= reach[:, None], -math.inf)
    p = torch.softmax(s, -1) if k.shape[0] else s
    return torch.where((reach > 0)[:, None], torch.nan_to_num(p) @ v, torch.zeros_like(q))


def _exact_append(x, cache, scales, table, starts, lens):
    """Block after block: scales are held in 32 bits, everything else in 64."""
    x, cache, scales = x.cpu().numpy().astype(np.float64), cache.cpu().numpy().astype(np.float64), \
        scales.cpu().numpy().astype(np.float32)
    bt = cache.shape[2]
    for b in range(len(lens)):
        rows = x[starts[b]:starts[b + 1]]
        at = int(lens[b]) - len(rows)
        i = 0
        while i < len(rows):
            off, blk = (at + i) % bt, table[b, (at + i) // bt]
            part = rows[i:i + bt - off].transpose(1, 0, 2)  # [heads, rows, dim]
            before = scales[blk] if off else np.zeros_like(scales[blk])
            scale = np.maximum(before, (np.abs(part).max((1, 2)) / 127.0).astype(np.float32))
            inv = np.zeros_like(scale)
            np.divide(np.float32(1), scale, out=inv, where=scale > 0)
            more = scale != before
            ratio = (before * inv).astype(np.float64)
            kept = np.rint(cache[blk, :, :off] * ratio[:, None, None])
            cache[blk, :, :off] = np.where(more[:, None, None], kept, cache[blk, :, :off])
            cache[blk, :, off:off + part.shape[1]] = np.rint(part * inv.astype(np.float64)[:, None, None])
            scales[blk] = scale
            i += part.shape[1]
    return cache, scales


def exact(case, seed):
    t = _inputs(case, seed)
    past, new = _lengths(case)
    total = past + new
    kvh, g, hd = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"]
    if case["op"] == "packed":
        out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
        qs, ks = _starts(new), _starts(total)
        for b in range(case["batch"]):
            reach = torch.arange(int(past[b]) + 1, int(total[b]) + 1, device="cuda")
            for h in range(case["q_heads"]):
                k, v = (t[n][ks[b]:ks[b + 1], h // g].double() for n in ("k", "v"))
                out[qs[b]:qs[b + 1], h] = _attend(t["q"][qs[b]:qs[b + 1], h].double(), k, v, reach)
        return out
    table, bt = t["block_tables"].cpu().numpy(), case["block"]
    if case["op"] == "append":
        starts, lens = t["seq_starts"].cpu().numpy(), t["seq_lens"].cpu().numpy()
        for n in ("k", "v"):
            cache, scales = _exact_append(t[n + "_new"], t[n + "_cache"], t[n + "_scales"], table,
                                          starts, lens)
            t[n + "_cache"], t[n + "_scales"] = torch.from_numpy(cache).cuda(), \
                torch.from_numpy(scales).cuda()

    def rows(name, b):  # [length, kv_heads, head_dim]
        blk = torch.from_numpy(table[b, :-(-int(total[b]) // bt)]).long().cuda()
        x = t[name + "_cache"][blk].double() * t[name + "_scales"][blk].double()[..., None, None]
        return x.permute(0, 2, 1, 3).reshape(-1, kvh, hd)[:int(total[b])]

    if case["op"] != "decode":
        return tuple(torch.cat([rows(n, b) for b in range(case["batch"])]) for n in ("k", "v"))
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        k, v = rows("k", b), rows("v", b)
        for h in range(kvh):
            heads = slice(h * g, (h + 1) * g)
            reach = torch.full((g,), int(total[b]), device="cuda")
            out[b, heads] = _attend(t["q"][b, heads].double(), k[:, h], v[:, h], reach)
    return out
