"""CPU tests of the 8-bit KV cache operators and the packed prompt
attention: argument rules of the C entry points (they return before any
launch), the wrappers' refusals, and the definition that the GPU tests use."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from mote_b200 import _native, errors, ops
from mote_b200.types import DType, plain
from tests import _q8_cache as ref

P, S = 0x1000, 0x2000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def append(lib, ptrs=(P,) * 9, tokens=1, batch=1, kvh=2, hd=64, blocks=4, bt=16, width=2, stream=S):
    return lib.mote_cuda_kv_cache_append_q8(*ptrs, tokens, batch, kvh, hd, blocks, bt, width, None,
                                            stream)


def read(lib, ptrs=(P,) * 8, tokens=1, batch=1, kvh=2, hd=64, blocks=4, bt=16, width=2, stream=S):
    return lib.mote_cuda_kv_cache_read_q8(*ptrs, tokens, batch, kvh, hd, blocks, bt, width, None,
                                          stream)


def decode(lib, ptrs=(P,) * 8, batch=1, qh=8, kvh=2, hd=64, blocks=4, bt=16, width=2, scale=0.1,
           ws=None, ws_bytes=0, stream=S):
    return lib.mote_cuda_gqa_attention_decode_q8(*ptrs, batch, qh, kvh, hd, blocks, bt, width,
                                                 scale, ws, ws_bytes, stream)


def packed(lib, ptrs=(P,) * 6, tokens=1, kv=1, batch=1, qh=8, kvh=2, hd=64, scale=0.1, stream=S):
    return lib.mote_cuda_gqa_attention_packed_f16(*ptrs, tokens, kv, batch, qh, kvh, hd, scale,
                                                  stream)


@pytest.mark.parametrize("call,n", [(append, 9), (read, 8), (decode, 8), (packed, 6)])
def test_null_and_unaligned_pointers(lib, call, n):
    for i in range(n):
        ptrs = [P] * n
        ptrs[i] = None
        assert call(lib, ptrs) == 1
        ptrs[i] = P + 2
        assert call(lib, ptrs) == 1
    assert call(lib, stream=None) == 1


@pytest.mark.parametrize("call", [append, read, decode])
def test_cache_shapes(lib, call):
    for bad in ({"hd": 96}, {"hd": 0}, {"bt": 8}, {"bt": 24}, {"bt": 0}, {"bt": 272},
                {"kvh": 65536}, {"batch": (1 << 20) + 1}, {"blocks": 1 << 31},
                {"width": (1 << 31) // 16}):
        assert call(lib, **bad) == 1, bad


def test_empty_calls(lib):
    assert append(lib, tokens=0) == 0 and append(lib, batch=0) == 0 and append(lib, kvh=0) == 0
    assert read(lib, tokens=0) == 0 and read(lib, batch=0) == 0
    assert decode(lib, batch=0) == 0 and decode(lib, qh=0) == 0
    assert packed(lib, tokens=0) == 0 and packed(lib, batch=0) == 0 and packed(lib, qh=0) == 0
    assert append(lib, tokens=1 << 31) == 1 and read(lib, tokens=1 << 31) == 1


def test_attention_arguments(lib):
    for call in (decode, packed):
        assert call(lib, qh=9) == 1 and call(lib, kvh=0) == 1 and call(lib, hd=96) == 1
        assert call(lib, qh=65536) == 1
        for scale in (float("nan"), float("inf")):
            assert call(lib, scale=scale) == 1
    # more units of work than 31 bits count, at the tables' full length
    assert decode(lib, batch=65535, qh=64, kvh=8, width=1 << 22) == 1
    assert packed(lib, scale=0.0) == 1 and packed(lib, scale=-1.0) == 1
    assert packed(lib, qh=258, kvh=2) == 1  # 129 query heads to a KV head
    assert packed(lib, tokens=1 << 31) == 1 and packed(lib, kv=1 << 31) == 1
    assert lib.mote_cuda_gqa_attention_decode_q8_workspace_bytes(1, 8, 2, 64, None) == 1


class _Context:
    """Stands where a refused call must not reach the device."""

    def storage(self, tensor):
        raise AssertionError("not refused")


class _Storage:
    pass


class _Tensor:
    def __init__(self, shape, dtype):
        self.desc = plain(shape, dtype)
        self.storage = _Storage()

    shape = property(lambda self: self.desc.shape)

    def shares_storage_with(self, other):
        return self.storage is other.storage


def tensors():
    return {"k_new": _Tensor((3, 2, 64), DType.F16), "v_new": _Tensor((3, 2, 64), DType.F16),
            "k_cache": _Tensor((4, 2, 16, 64), DType.I8),
            "v_cache": _Tensor((4, 2, 16, 64), DType.I8),
            "k_scales": _Tensor((4, 2), DType.F32), "v_scales": _Tensor((4, 2), DType.F32),
            "block_tables": _Tensor((1, 2), DType.I32), "seq_starts": _Tensor((2,), DType.I32),
            "seq_lens": _Tensor((1,), DType.I32), "q": _Tensor((1, 8, 64), DType.F16),
            "output": _Tensor((1, 8, 64), DType.F16)}


CACHE = ("k_cache", "v_cache", "k_scales", "v_scales", "block_tables")
OPS = {"append": (ops.kv_cache_append_q8, ("k_new", "v_new", *CACHE, "seq_starts", "seq_lens")),
       "read": (ops.kv_cache_read_q8, (*CACHE, "seq_starts", "k_new", "v_new")),
       "decode": (ops.gqa_attention_decode_q8, ("q", *CACHE, "seq_lens", "output"))}


@pytest.mark.parametrize("op", list(OPS))
def test_wrappers_refuse(op):
    fn, names = OPS[op]

    def call(**other):
        t = tensors() | other
        fn(_Context(), *(t[n] for n in names))

    with pytest.raises(AssertionError):
        call()  # everything fits: it goes on to the storages
    for name in names:
        desc = tensors()[name].desc
        wrong = DType.F16 if desc.encoding.plain is not DType.F16 else DType.F32
        with pytest.raises(errors.DTypeMismatch):
            call(**{name: _Tensor(desc.shape, wrong)})
        with pytest.raises((errors.ShapeMismatch, errors.RankMismatch)):
            call(**{name: _Tensor((*desc.shape, 1), desc.encoding.plain)})
        with pytest.raises((errors.ShapeMismatch, errors.RankMismatch, AssertionError)) as e:
            call(**{name: _Tensor((desc.shape[0] + 1, *desc.shape[1:]), desc.encoding.plain)})
        # one more block or sequence than the others say
        assert e.type is not AssertionError or (op == "read" and name == "seq_lens")
    t = tensors()
    pair = {"append": ("k_cache", "v_cache"), "read": ("k_new", "v_new"),
            "decode": ("q", "output")}[op]
    t[pair[1]] = t[pair[0]]
    with pytest.raises(errors.AliasedStorage):
        fn(_Context(), *(t[n] for n in names))


def test_packed_wrapper_refuses():
    def t():
        return {"q": _Tensor((5, 8, 64), DType.F16), "k": _Tensor((9, 2, 64), DType.F16),
                "v": _Tensor((9, 2, 64), DType.F16), "q_starts": _Tensor((3,), DType.I32),
                "kv_starts": _Tensor((3,), DType.I32), "output": _Tensor((5, 8, 64), DType.F16)}

    def call(**other):
        ops.gqa_attention_packed_f16(_Context(), *(t() | other).values())

    with pytest.raises(AssertionError):
        call()
    for name, desc in ((n, x.desc) for n, x in t().items()):
        wrong = DType.F32 if desc.encoding.plain is not DType.F32 else DType.F16
        with pytest.raises(errors.DTypeMismatch):
            call(**{name: _Tensor(desc.shape, wrong)})
        with pytest.raises((errors.ShapeMismatch, errors.RankMismatch)):
            call(**{name: _Tensor((*desc.shape, 1), desc.encoding.plain)})
    for other in ({"k": _Tensor((9, 2, 128), DType.F16)}, {"v": _Tensor((8, 2, 64), DType.F16)},
                  {"kv_starts": _Tensor((4,), DType.I32)}, {"q_starts": _Tensor((0,), DType.I32)}):
        with pytest.raises(errors.ShapeMismatch):
            call(**other)
    x = t()
    for name in ("q", "k", "v"):
        if x[name].shape == x["output"].shape:
            with pytest.raises(errors.AliasedStorage):
                call(**{name: x["output"], "output": x["output"]})


def test_definition_of_the_append():
    """A block by hand: scale, ties to even, rounding again as it grows."""
    cache, scales = np.full((1, 1, 16, 64), 9, np.int8), np.full((1, 1), 5, np.float32)
    x = np.zeros((2, 1, 64), np.float16)
    x[0, 0, :4] = [127, 63.5, -63.5, 0.25]
    x[1, 0, 0] = 1.5
    ref.append(cache, scales, [[0]], x, [2], [0, 2])
    assert scales[0, 0] == 1
    assert cache[0, 0, 0, :4].tolist() == [127, 64, -64, 0] and cache[0, 0, 1, 0] == 2
    assert (cache[0, 0, 2:] == 9).all()
    x = np.full((1, 1, 64), 254, np.float16)
    ref.append(cache, scales, [[0]], x, [3], [0, 1])
    assert scales[0, 0] == 2 and cache[0, 0, 0, :3].tolist() == [64, 32, -32]
    assert cache[0, 0, 1, 0] == 1 and (cache[0, 0, 2] == 127).all()


def test_rounding_by_a_sum_is_rint():
    """fl32(x * m + 1.5 * 2^23) holds rint(x * m), |x * m| <= 128, whatever m:
    the exact sum is rounded once, to a multiple of 1."""
    r = np.random.default_rng(1)
    x = r.normal(0, 1, 200000).astype(np.float16)
    m = (127 / np.abs(x.astype(np.float64)).max() * r.uniform(0.5, 1, x.size)).astype(np.float32)
    exact = x.astype(np.float64) * m.astype(np.float64)
    ties = np.float64(0.5) + np.arange(-128, 128)
    exact = np.concatenate([exact, ties])
    got = (exact + 12582912.0).astype(np.float32).view(np.int32).astype(np.int64) - \
        np.float32(12582912.0).view(np.int32)
    # one rounding in the device's fma; here the 64-bit sum adds none: 35 + 9 bits fit
    assert np.array_equal(got, np.rint(exact).astype(np.int64))


def test_ctypes_arity():
    for name, n in (("kv_cache_append_q8", 18), ("kv_cache_read_q8", 17),
                    ("gqa_attention_decode_q8", 19), ("gqa_attention_packed_f16", 14)):
        assert len(_native.SIGNATURES["mote_cuda_" + name][1]) == n
    assert ctypes.sizeof(_native.P) == 8
