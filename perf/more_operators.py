"""Measured cases of the paged f16 KV cache and of what stands around it.

Three operators that a decoder layer calls one after another:

* ``axes``: the cos/sin tables of rotary positions with several axes (time,
  height, width);
* ``append``: the rows of a fused QKV projection, rotated by those tables, q
  to its own buffer, k and v into the pages of their sequences;
* ``attn``: the new tokens of every sequence (one, a few, a chunk of a prompt,
  or a mix of these) over the pages, causal, grouped-query.

Head layouts are 32 query / 8 KV heads with head_dim 64 and 128 (this
repository's decoder layers) and the extremes of the grouping.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------- cases --
def _axes(name, tokens, s0, s1, s2, order, theta):
    return {"name": name, "op": "axes", "tokens": tokens, "s0": s0, "s1": s1, "s2": s2,
            "order": order, "theta": theta}


def _paged(name, op, lens, batch, lo, hi, past_lo=0, past_hi=0, single=0, q_heads=32, kv_heads=8,
           head_dim=128, block=32, pairs=64, layout="half"):
    c = {"name": name, "op": op, "lens": lens, "batch": batch, "single": single, "lo": lo,
         "hi": hi, "past_lo": past_lo, "past_hi": past_hi, "q_heads": q_heads,
         "kv_heads": kv_heads, "head_dim": head_dim, "block": block}
    return c | ({"pairs": pairs, "layout": layout} if op == "append" else {})


def listed():
    return [
        # one prompt with a picture in it
        _axes("axes_picture", 1237, 16, 24, 24, "sections", 1e6),
        # a long video, pairs dealt to the axes in turn
        _axes("axes_video", 65536, 24, 20, 20, "interleaved", 5e5),
        # one new token for each of 32 running sequences
        _paged("append_step", "append", 1, 32, 1, 1, 20, 4000, block=16),
        # whole prompts of a batch written at once
        _paged("append_prompts", "append", 2, 16, 40, 2048, 0, 90),
        # one user, short context: latency
        _paged("decode_one_short", "attn", 3, 1, 1, 1, 116, 116, head_dim=64, block=16),
        # one user, long context: the split over positions and its join
        _paged("decode_one_long", "attn", 4, 1, 1, 1, 32767, 32767, block=64),
        # a serving batch whose lengths differ by orders of magnitude
        _paged("decode_ragged", "attn", 5, 48, 1, 1, 0, 8191, block=16),
        # a few drafted tokens of each sequence looked over at once
        _paged("verify_few", "attn", 6, 16, 3, 8, 500, 4000),
        # running sequences with a chunk of a new prompt among them
        _paged("step_mixed", "attn", 7, 33, 512, 512, 100, 4000, single=32, head_dim=64, block=64),
        # chunks of several prompts, 1B-sized heads
        _paged("chunks_d64", "attn", 8, 6, 300, 1024, 0, 2500, head_dim=64),
        # a short question on a long document that is cached already
        _paged("question_long", "attn", 9, 1, 61, 61, 32000, 32000, block=128),
        # a chunk of a very long prompt: the largest
        _paged("chunk_long", "attn", 10, 1, 2048, 2048, 16384, 16384),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


MOST_PAIRS = 32 * 128 * 2048 * (16384 + 1024)  # query heads x head_dim x attended positions, largest case
MOST_SCORES = 1 << 31  # of a padded batch
MOST_ROWS = 200000     # cached positions of a batch


def draw(rng):
    op = rng.choice(["axes", "append", "append", "attn", "attn", "attn", "attn", "attn"])
    if op == "axes":
        s = [rng.randint(1, 24) for _ in range(3)]
        order = rng.choice(["sections", "interleaved", "own"])
        if order == "interleaved":  # as many pairs of axis 0 as the others need between them
            s[0] = max(1, 3 * max(s[1:]) - s[1] - s[2]) + rng.randint(0, 8)
        return {"op": op, "tokens": _log_int(rng, 1, 65536), "s0": s[0], "s1": s[1], "s2": s[2],
                "order": order, "theta": rng.choice([1e4, 5e5, 1e6])}
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16] if kv_heads < 8 else [1, 2, 4, 5])
    c = {"op": op, "lens": rng.randrange(1, 1 << 30), "q_heads": kv_heads * group,
         "kv_heads": kv_heads, "head_dim": head_dim, "block": rng.choice([16, 32, 48, 64, 128, 256])}
    if op == "append":
        hi = _log_int(rng, 1, 2048)
        batch = _log_int(rng, 1, min(64, 15000 // hi))
        past = rng.choice([0, _log_int(rng, 1, 1000)])
        return c | {"batch": batch, "single": 0, "lo": rng.randint(0 if batch > 1 else 1, hi), "hi": hi,
                    "past_lo": 0, "past_hi": past, "pairs": rng.choice([head_dim // 2, head_dim // 4, 8]),
                    "layout": rng.choice(["half", "interleaved"])}
    kind = rng.choice(["decode", "few", "chunk", "mixed"])
    hi = {"decode": 1, "few": rng.randint(2, 16)}.get(kind) or _log_int(rng, 17, 2048)
    past = _log_int(rng, 1, 32768)
    per = c["q_heads"] * head_dim
    past = min(past, max(1, MOST_PAIRS // (per * hi) - hi // 2), MOST_SCORES // (c["q_heads"] * hi) - hi)
    batch = _log_int(rng, 1, max(1, min(
        1 if kind == "mixed" else 64, MOST_ROWS // (past + hi), MOST_PAIRS // (per * hi * (past + hi)),
        MOST_SCORES // (c["q_heads"] * hi * (past + hi)))))
    single = 0
    if kind == "mixed":
        single = _log_int(rng, 1, max(1, min(32, MOST_ROWS // (past + hi) - 1,
                                             MOST_SCORES // (c["q_heads"] * hi * (past + hi)) - 1)))
    lo = hi if kind in ("decode", "mixed") else rng.randint(0 if batch > 1 else 1, hi)
    return c | {"batch": batch + single, "single": single, "lo": lo, "hi": hi,
                "past_lo": rng.choice([0, past // 2, past]), "past_hi": past}


def _lengths(case):
    """(past, new) lengths of the sequences: [batch] each."""
    r = np.random.RandomState(case["lens"])
    new = r.randint(case["lo"], case["hi"] + 1, case["batch"]).astype(np.int64)
    new[r.randint(case["batch"])] = case["hi"]
    if case["single"]:
        new[:] = 1
        new[r.permutation(case["batch"])[case["single"]:]] = case["hi"]
    past = r.randint(case["past_lo"], case["past_hi"] + 1, case["batch"]).astype(np.int64)
    return past, new


def _starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def work(case):
    if case["op"] == "axes":
        pairs = case["s0"] + case["s1"] + case["s2"]
        return {"bytes": case["tokens"] * (12 + 8 * pairs), "flops": 4 * case["tokens"] * pairs}
    past, new = _lengths(case)
    qh, kvh, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    total, tokens = past + new, int(new.sum())
    if case["op"] == "append":
        held = 4 * int((-(-total // case["block"]) - past // case["block"]).sum()) + 8 * case["batch"]
        return {"bytes": tokens * ((qh + 2 * kvh) * hd * 4 + case["pairs"] * 8) + held,
                "flops": 6 * tokens * (qh + kvh) * case["pairs"]}
    attended = total[new > 0]
    held = 4 * int((-(-attended // case["block"])).sum()) + 8 * case["batch"]
    pairs = int((new * past + new * (new + 1) // 2).sum())
    return {"bytes": 4 * kvh * hd * int(attended.sum()) + 4 * qh * hd * tokens + held,
            "flops": 4 * hd * qh * pairs}


# ------------------------------------------------------------------ inputs --
def _gains(gen, heads, head_dim):
    """Channel gains of K: a few channels stand out, as keys' do."""
    g = torch.ones(heads, 1, head_dim, device="cuda", dtype=torch.float16)
    g[:, :, torch.randint(0, head_dim, (2,), generator=gen, device="cuda")] = 4.0
    return g


def _grid_positions(tokens, r):
    """Positions [3, tokens] of text with pictures (frames) between: text
    moves all axes, a picture's patches count rows and columns."""
    out, at, n = [], int(r.randint(0, 50)), 0
    while n < tokens:
        text = int(r.randint(1, 40))
        out.append(np.arange(at, at + text)[None].repeat(3, 0))
        at += text
        h, w = int(r.randint(4, 40)), int(r.randint(4, 40))
        grid = np.zeros((3, h, w), np.int64) + at
        grid[1] += np.arange(h)[:, None]
        grid[2] += np.arange(w)
        out.append(grid.reshape(3, -1))
        at += max(h, w)
        n += text + h * w
    return np.concatenate(out, 1)[:, :tokens].astype(np.int32)


def _inputs(case, seed):
    """The case's tensors from the seed, on the GPU."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 13)
    r = np.random.RandomState((int(seed) * 31 + 5) % (1 << 31))

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)

    if case["op"] == "axes":
        return {"positions": ints(_grid_positions(case["tokens"], r))}
    past, new = _lengths(case)
    total = past + new
    qh, kvh, hd, bt, batch = (case[n] for n in ("q_heads", "kv_heads", "head_dim", "block", "batch"))
    need = -(-total // bt)
    num_blocks = int(need.sum()) + 3
    # pages in no order, unused table entries -1
    order = r.permutation(num_blocks)
    table = np.full((batch, max(1, int(need.max()))), -1, np.int32)
    at = _starts(need)
    for b in range(batch):
        table[b, :need[b]] = order[at[b]:at[b + 1]]
    t = {"block_tables": ints(table), "seq_lens": ints(total), "starts": ints(_starts(new)),
         "k_cache": randn(num_blocks, kvh, bt, hd).mul_(_gains(gen, kvh, hd)),
         "v_cache": randn(num_blocks, kvh, bt, hd)}
    tokens = int(new.sum())
    if case["op"] == "attn":
        t["q"] = randn(tokens, qh, hd)
        return t
    t["qkv"] = randn(tokens, qh + 2 * kvh, hd)
    position = torch.from_numpy(np.concatenate([np.arange(p, p + n) for p, n in zip(past, new)])).cuda()
    angle = position[:, None].double() * 500000.0 ** (
        -torch.arange(case["pairs"], device="cuda").double() / case["pairs"])
    t["cos"], t["sin"] = angle.cos().float(), angle.sin().float()
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
             torch.int32: (types.DType.I32, "<i4")}
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
    if case["op"] == "axes":
        shape = (case["tokens"], case["s0"] + case["s1"] + case["s2"])
        outs = {n: torch.zeros(shape, device="cuda") for n in ("cos", "sin")}
        most = 0
    else:
        past, new = _lengths(case)
        most = int(new.max())  # a serving program knows its lengths
        rows = (int(new.sum()), case["q_heads"], case["head_dim"])
        outs = {"out": torch.zeros(rows, dtype=torch.float16, device="cuda")}
    state = {"case": case, "in": t, "most": most}
    if own:
        state["held"], state["seen"] = _framework_tensors(t | outs)
        state["in"] = None
        state["context"] = _context
    return state


# ------------------------------------------------------------- plain forms --
def _pair_axes(case):
    """(axis, exponent of 1 / theta) of every pair."""
    s = [case["s0"], case["s1"], case["s2"]]
    pairs = sum(s)
    j = np.arange(pairs)
    axis = np.repeat(np.arange(3), s)
    if case["order"] == "interleaved":
        axis = np.where(j // 3 < np.asarray(s)[j % 3], j % 3, 0)
    if case["order"] == "own":
        return axis, np.concatenate([np.arange(n) / n for n in s])
    return axis, j / pairs


def _plain_axes(case, t):
    axis, exponent = (torch.from_numpy(a).to(t["positions"].device) for a in _pair_axes(case))
    angle = t["positions"][axis].T.double() * case["theta"] ** -exponent
    return angle.cos().float(), angle.sin().float()


def _rows(starts, count):
    """(sequence, index in it) of each of `count` packed rows."""
    row = torch.arange(count, device=starts.device)
    seq = torch.searchsorted(starts[1:].contiguous(), row.int(), right=True)
    return seq, row - starts[seq]


def _plain_append(case, t):
    qkv, cos, sin = t["qkv"], t["cos"][:, None], t["sin"][:, None]
    qh, kvh, pairs = case["q_heads"], case["kv_heads"], case["pairs"]
    qk = qkv[:, :qh + kvh].float()
    out = qk.clone()
    if case["layout"] == "half":
        a, b = slice(0, pairs), slice(pairs, 2 * pairs)
    else:
        a, b = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
    out[..., a] = qk[..., a] * cos - qk[..., b] * sin
    out[..., b] = qk[..., b] * cos + qk[..., a] * sin
    out = out.half()
    k_cache, v_cache, bt = t["k_cache"], t["v_cache"], case["block"]
    seq, idx = _rows(t["starts"], qkv.shape[0])
    new = t["starts"][1:] - t["starts"][:-1]
    pos = (t["seq_lens"] - new)[seq] + idx
    block, off = t["block_tables"][seq, pos // bt].long(), pos % bt
    k_cache[block, :, off] = out[:, qh:]
    v_cache[block, :, off] = qkv[:, qh + kvh:]
    return out[:, :qh].contiguous(), k_cache, v_cache


def _plain_attn(t, most):
    q, starts, lens = t["q"], t["starts"], t["seq_lens"]
    table = t["block_tables"].clamp(min=0).long()
    qh, hd = q.shape[1:]
    kvh, batch = t["k_cache"].shape[1], lens.numel()

    def padded(name):  # [batch, kv_heads, 1, positions, head_dim]
        c = t[name][table].float()
        return c.permute(0, 2, 1, 3, 4).reshape(batch, kvh, 1, -1, hd)

    seq, idx = _rows(starts, q.shape[0])
    pq = torch.zeros(batch, most, qh, hd, device=q.device)
    pq[seq, idx] = q.float() * (1.0 / math.sqrt(hd))
    pq = pq.view(batch, most, kvh, qh // kvh, hd).permute(0, 2, 3, 1, 4)
    k = padded("k_cache")
    scores = torch.matmul(pq, k.transpose(-1, -2))
    del pq
    past = lens - (starts[1:] - starts[:-1])
    last = past.view(-1, 1) + torch.arange(most, device=q.device)
    hidden = torch.arange(k.shape[3], device=q.device) > last.unsqueeze(-1)
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    e = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(e, padded("v_cache")).div_(e.sum(-1, keepdim=True))
    return out.permute(0, 3, 1, 2, 4).reshape(batch, most, qh, hd)[seq, idx].half()


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from mote_b200 import ops, types

        c, h, seen = state["context"], state["held"], state["seen"]
        if op == "axes":
            order = {"sections": types.RopeAxes.Sections, "interleaved": types.RopeAxes.Interleaved,
                     "own": types.RopeAxes.Own}[case["order"]]
            ops.rope_cos_sin_axes_f32(c, h["positions"], h["cos"], h["sin"],
                                      (case["s0"], case["s1"], case["s2"]), case["theta"], order)
            return seen["cos"], seen["sin"]
        if op == "append":
            layout = {"half": types.RopeLayout.HalfSplit,
                      "interleaved": types.RopeLayout.Interleaved}[case["layout"]]
            ops.rope_kv_cache_append_paged_f16(c, h["qkv"], h["cos"], h["sin"], h["out"],
                                               h["k_cache"], h["v_cache"], h["block_tables"],
                                               h["starts"], h["seq_lens"], layout, check=False)
            return seen["out"], seen["k_cache"], seen["v_cache"]
        ops.gqa_attention_paged_f16(c, h["q"], h["k_cache"], h["v_cache"], h["block_tables"],
                                    h["starts"], h["seq_lens"], h["out"], state["most"])
        return seen["out"]
    t = state["in"]
    if op == "axes":
        return _plain_axes(case, t)
    return _plain_append(case, t) if op == "append" else _plain_attn(t, state["most"])


# ---------------------------------------------- the definitions in 64 bits --
def _exact_axes(case, t):
    p = t["positions"].cpu().numpy().astype(np.float64)
    s = [case["s0"], case["s1"], case["s2"]]
    pairs, angles, used = sum(s), [], [0, 0, 0]
    for j in range(pairs):
        if case["order"] == "interleaved":
            axis = j % 3 if j // 3 < s[j % 3] else 0
        else:
            axis = 0 if j < s[0] else 1 if j < s[0] + s[1] else 2
        power = used[axis] / s[axis] if case["order"] == "own" else j / pairs
        used[axis] += 1
        angles.append(torch.from_numpy(p[axis] / math.pow(case["theta"], power)))
    angles = torch.stack(angles, 1)
    return torch.cos(angles), torch.sin(angles)


def _exact_append(case, t):
    qh, kvh, pairs, bt = case["q_heads"], case["kv_heads"], case["pairs"], case["block"]
    rows = t["qkv"].double()
    turn = torch.complex(t["cos"].double(), t["sin"].double())[:, None]
    x = rows[:, :qh + kvh, :2 * pairs]
    x = x.unflatten(-1, (2, pairs)).transpose(-1, -2) if case["layout"] == "half" else x.unflatten(-1, (pairs, 2))
    y = torch.view_as_real(torch.view_as_complex(x.contiguous()) * turn)
    y = (y.transpose(-1, -2) if case["layout"] == "half" else y).flatten(-2)
    rows[:, :qh + kvh, :2 * pairs] = y
    past, new = _lengths(case)
    table, starts = t["block_tables"].cpu().numpy(), _starts(new)
    k_cache, v_cache = t["k_cache"].double(), t["v_cache"].double()
    for b in range(case["batch"]):
        at = int(past[b])
        while at < past[b] + new[b]:
            n = min(bt - at % bt, int(past[b] + new[b]) - at)
            first = int(starts[b]) + at - int(past[b])
            part = rows[first:first + n].transpose(0, 1)
            here = (int(table[b, at // bt]), slice(None), slice(at % bt, at % bt + n))
            k_cache[here], v_cache[here] = part[qh:qh + kvh], part[qh + kvh:]
            at += n
    return rows[:, :qh], k_cache, v_cache


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "axes":
        return _exact_axes(case, t)
    if case["op"] == "append":
        return _exact_append(case, t)
    past, new = _lengths(case)
    kvh, g, hd, bt = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"], case["block"]
    starts, out = _starts(new), torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n, total = int(new[b]), int(past[b] + new[b])
        if n == 0:
            continue
        blocks = t["block_tables"][b, :-(-total // bt)].long()
        hidden = torch.triu(torch.ones(n, total, dtype=torch.bool, device="cuda"), int(past[b]) + 1)
        for h in range(kvh):
            k, v = (t[c][blocks, h].reshape(-1, hd)[:total].double() for c in ("k_cache", "v_cache"))
            for j in range(h * g, (h + 1) * g):
                q = t["q"][int(starts[b]):int(starts[b]) + n, j].double()
                s = ((q @ k.T) / math.sqrt(hd)).masked_fill(hidden, -math.inf)
                out[int(starts[b]):int(starts[b]) + n, j] = torch.softmax(s, -1) @ v
    return out
