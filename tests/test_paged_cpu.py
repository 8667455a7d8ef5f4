"""CPU tests of the paged f16 cache's operators: argument rules of the C entry
points (they return before any launch) and the wrappers' refusals."""
from __future__ import annotations

import itertools

import pytest

from mote_b200 import _native, errors, ops
from mote_b200.types import DType, RopeAxes
from tests.test_q8_cache_cpu import _Context, _Tensor

P, S = 0x1000, 0x2000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def axes(lib, ptrs=(P,) * 3, tokens=1, n=3, s=(16, 24, 24, 0), order=0, theta=1e4, stream=S):
    return lib.mote_cuda_rope_cos_sin_axes_f32(*ptrs, tokens, n, *s, order, theta, stream)


def append(lib, ptrs=(P,) * 9, tokens=1, batch=1, qh=8, kvh=2, hd=64, pairs=32, blocks=4, bt=16,
           width=2, layout=0, flag=None, stream=S):
    return lib.mote_cuda_rope_kv_cache_append_paged_f16(*ptrs, tokens, batch, qh, kvh, hd, pairs,
                                                        blocks, bt, width, layout, flag, stream)


def attend(lib, ptrs=(P,) * 7, tokens=1, batch=1, qh=8, kvh=2, hd=64, blocks=4, bt=16, width=2,
           most=1, scale=0.1, ws=None, ws_bytes=0, stream=S):
    return lib.mote_cuda_gqa_attention_paged_f16(*ptrs, tokens, batch, qh, kvh, hd, blocks, bt,
                                                 width, most, scale, ws, ws_bytes, stream)


@pytest.mark.parametrize("call,n", [(axes, 3), (append, 9), (attend, 7)])
def test_null_and_unaligned_pointers(lib, call, n):
    for i in range(n):
        ptrs = [P] * n
        ptrs[i] = None
        assert call(lib, ptrs) == 1
        ptrs[i] = P + 2
        assert call(lib, ptrs) == 1
    assert call(lib, stream=None) == 1


def test_append_without_rotation_takes_no_tables(lib):
    ptrs = [P, None, None] + [P] * 6
    assert append(lib, ptrs, pairs=0, tokens=0) == 0
    assert append(lib, ptrs, pairs=1, tokens=0) == 1


@pytest.mark.parametrize("call", [append, attend])
def test_cache_shapes(lib, call):
    for bad in ({"hd": 96}, {"hd": 0}, {"hd": 256}, {"bt": 8}, {"bt": 24}, {"bt": 0}, {"bt": 272},
                {"kvh": 65536}, {"batch": (1 << 20) + 1}, {"blocks": 1 << 31},
                {"width": (1 << 31) // 16}, {"tokens": 1 << 31}, {"qh": 65536}):
        assert call(lib, **bad) == 1, bad


def test_append_values(lib):
    for bad in ({"pairs": 33}, {"pairs": 1 << 63}, {"layout": 2}, {"flag": P + 2}):
        assert append(lib, **bad) == 1, bad
    assert append(lib, tokens=0) == 0
    assert append(lib, batch=0) == 0


def test_attention_values(lib):
    for bad in ({"qh": 7}, {"kvh": 0}, {"qh": 258, "kvh": 2}, {"scale": 0.0}, {"scale": -1.0},
                {"scale": float("nan")}, {"scale": float("inf")}, {"most": 1 << 31}):
        assert attend(lib, **bad) == 1, bad
    assert attend(lib, tokens=0) == 0
    assert attend(lib, batch=0) == 0
    assert attend(lib, qh=0) == 0


def test_axes_values(lib):
    for bad in ({"n": 0}, {"n": 5}, {"order": 3}, {"theta": 0.5}, {"theta": float("nan")},
                {"theta": float("inf")}, {"s": (64, 64, 1, 0)}, {"n": 2}, {"tokens": 1 << 31},
                {"s": ((1 << 32) - 1, 2, 0, 0)},
                # the last pair of axis 1 would be number 1 + 3 * 9 of 21
                {"s": (10, 10, 1, 0), "order": 1}):
        assert axes(lib, **bad) == 1, bad
    assert axes(lib, tokens=0) == 0
    assert axes(lib, s=(0, 0, 0, 0)) == 0


def tensors():
    return {"qkv": _Tensor((5, 12, 64), DType.F16), "cos": _Tensor((5, 32), DType.F32),
            "sin": _Tensor((5, 32), DType.F32), "q_out": _Tensor((5, 8, 64), DType.F16),
            "k_cache": _Tensor((4, 2, 16, 64), DType.F16),
            "v_cache": _Tensor((4, 2, 16, 64), DType.F16),
            "block_tables": _Tensor((3, 2), DType.I32), "starts": _Tensor((4,), DType.I32),
            "seq_lens": _Tensor((3,), DType.I32)}


ATTEND = ("q_out", "k_cache", "v_cache", "block_tables", "starts", "seq_lens")


def run_append(t, **kw):
    ops.rope_kv_cache_append_paged_f16(_Context(), *t.values(), **kw)


def run_attend(t, most=5):
    ops.gqa_attention_paged_f16(_Context(), *(t[n] for n in ATTEND), t["output"], most)


@pytest.mark.parametrize("run", [run_append, run_attend])
@pytest.mark.parametrize("name", ["k_cache", "v_cache", "block_tables", "starts", "seq_lens",
                                  "q_out"])
def test_wrapper_names_the_wrong_operand(run, name):
    t = tensors()
    t["output"] = _Tensor((5, 8, 64), DType.F16)
    if run is run_append:
        del t["output"]
    shape = t[name].desc.shape
    for wrong, error in (((*shape, 1), errors.RankMismatch),
                         ((shape[0] + 1, *shape[1:]), errors.ShapeMismatch)):
        bad = dict(t) | {name: _Tensor(wrong, t[name].desc.encoding.plain)}
        with pytest.raises(error):
            run(bad)
    bad = dict(t) | {name: _Tensor(shape, DType.U8)}
    with pytest.raises(errors.CudaError):
        run(bad)


def test_append_outputs_share_no_storage():
    names = ("q_out", "k_cache", "v_cache")
    for a, b in [*itertools.combinations(names, 2), *((n, "qkv") for n in names)]:
        t = tensors()
        t[a].storage = t[b].storage
        with pytest.raises(errors.AliasedStorage):
            run_append(t)


@pytest.mark.parametrize("name", ["q_out", "k_cache", "v_cache"])
def test_attention_output_shares_no_storage(name):
    t = tensors()
    t["output"] = _Tensor((5, 8, 64), DType.F16)
    t["output"].storage = t[name].storage
    with pytest.raises(errors.AliasedStorage):
        run_attend(t)


def test_append_refuses_more_pairs_than_a_head_has():
    t = tensors()
    t["cos"], t["sin"] = _Tensor((5, 33), DType.F32), _Tensor((5, 33), DType.F32)
    with pytest.raises(errors.InvalidRotaryDim):
        run_append(t)


def test_attention_refuses_a_negative_count():
    t = tensors()
    t["output"] = _Tensor((5, 8, 64), DType.F16)
    with pytest.raises(errors.ShapeMismatch):
        run_attend(t, -1)


def test_axes_wrapper():
    pos, cos, sin = (_Tensor((3, 5), DType.I32), _Tensor((5, 64), DType.F32),
                     _Tensor((5, 64), DType.F32))
    run = ops.rope_cos_sin_axes_f32
    with pytest.raises(errors.ShapeMismatch):
        run(_Context(), pos, cos, sin, (32, 32))
    with pytest.raises(errors.ShapeMismatch):
        run(_Context(), pos, cos, sin, (16, 24, 23), order=RopeAxes.Own)
    with pytest.raises(errors.ShapeMismatch):
        run(_Context(), pos, cos, sin, (16, 49, -1))
    with pytest.raises(errors.AliasedStorage):
        run(_Context(), pos, cos, cos, (16, 24, 24))


def test_workspace_size_is_kept_by_what_it_depends_on(monkeypatch):
    """head_dim and the class of query rows, not the calls' sizes; a call that is
    refused leaves nothing behind."""
    import ctypes

    from mote_b200 import context

    asked = []

    class _Lib:
        @staticmethod
        def mote_cuda_gqa_attention_paged_f16_workspace_bytes(qh, kvh, hd, most, out):
            rows = most * (qh // kvh) if kvh else 0
            asked.append((hd, rows))
            ctypes.cast(out, ctypes.POINTER(ctypes.c_uint64))[0] = \
                (1000 * hd + (rows > 8) + (rows > 16)) if kvh and hd in (64, 128) else 0
            return 0

    class _Inner:
        def select(self):
            pass

    monkeypatch.setattr(context, "lib", lambda: _Lib)
    c = context.CudaContext.__new__(context.CudaContext)
    c.inner = _Inner()
    assert c.paged_workspace_bytes(8, 0, 64, 1) == 0
    assert c.paged_workspace_bytes(8, 2, 96, 1) == 0
    for most in range(1, 300):
        assert c.paged_workspace_bytes(8, 2, 64, most) == 64000 + (most > 2) + (most > 4)
        assert c.paged_workspace_bytes(32, 2, 128, most) == 128000 + 1 + (most > 1)
    assert len(c._paged_need) == 5 and len(asked) == 7


def test_workspace_size_follows_its_classes(lib):
    """The library's own sizes change at 8 and at 16 query rows and nowhere else
    (without a device every call fails alike)."""
    import ctypes

    def size(qh, kvh, hd, most):
        out = ctypes.c_uint64(0)
        status = lib.mote_cuda_gqa_attention_paged_f16_workspace_bytes(qh, kvh, hd, most, ctypes.byref(out))
        return status, out.value

    for hd in (64, 128):
        for a, b in (((8, 2, 1), (8, 2, 2)), ((8, 2, 3), (16, 1, 1)), ((8, 2, 5), (128, 1, 900))):
            assert size(a[0], a[1], hd, a[2]) == size(b[0], b[1], hd, b[2])
    assert size(0, 2, 64, 1) == (0, 0) and size(8, 0, 64, 1) == (0, 0) and size(8, 2, 96, 1) == (0, 0)
