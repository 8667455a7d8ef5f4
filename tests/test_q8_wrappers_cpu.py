"""CPU tests of the 8-bit cache's and the packed attention's wrappers: every
pair of tensors that must not share storage, the memo of the workspace's size
and the largest work list of a decode call."""
from __future__ import annotations

import ctypes

import pytest

from mote_b200 import _native, context, errors, ops
from mote_b200.types import DType
from tests.test_q8_cache_cpu import _Context, _Tensor, decode, tensors


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_packed_output_shares_no_storage(name):
    """One storage under two descriptors, whatever their shapes."""
    t = {"q": _Tensor((5, 8, 64), DType.F16), "k": _Tensor((9, 2, 64), DType.F16),
         "v": _Tensor((9, 2, 64), DType.F16), "q_starts": _Tensor((3,), DType.I32),
         "kv_starts": _Tensor((3,), DType.I32), "output": _Tensor((5, 8, 64), DType.F16)}
    t["output"].storage = t[name].storage
    with pytest.raises(errors.AliasedStorage):
        ops.gqa_attention_packed_f16(_Context(), *t.values())


@pytest.mark.parametrize("op,names,pairs", [
    (ops.kv_cache_append_q8, ("k_new", "v_new", "k_cache", "v_cache", "k_scales", "v_scales",
                              "block_tables", "seq_starts", "seq_lens"),
     [("k_cache", "v_cache"), ("k_scales", "v_scales")]),
    (ops.kv_cache_read_q8, ("k_cache", "v_cache", "k_scales", "v_scales", "block_tables",
                            "seq_starts", "k_new", "v_new"), [("k_new", "v_new")]),
    (ops.gqa_attention_decode_q8, ("q", "k_cache", "v_cache", "k_scales", "v_scales",
                                   "block_tables", "seq_lens", "output"), [("q", "output")])])
def test_cache_outputs_share_no_storage(op, names, pairs):
    for a, b in pairs:
        t = tensors()
        t[a].storage = t[b].storage
        with pytest.raises(errors.AliasedStorage):
            op(_Context(), *(t[n] for n in names))


def test_workspace_size_is_kept_by_head_dim(monkeypatch):
    """Not by batch, and a call without work or of another head_dim leaves
    nothing behind that a later call would take."""
    asked = []

    class _Lib:
        @staticmethod
        def mote_cuda_gqa_attention_decode_q8_workspace_bytes(b, qh, kvh, hd, out):
            asked.append(hd)
            found = hd in (64, 128) and b and qh and kvh
            ctypes.cast(out, ctypes.POINTER(ctypes.c_uint64))[0] = 1000 * hd if found else 0
            return 0

    monkeypatch.setattr(context, "lib", lambda: _Lib)

    class _Inner:
        def select(self):
            pass

    c = context.CudaContext.__new__(context.CudaContext)
    c.inner = _Inner()
    assert c.decode_q8_workspace_bytes(0, 0, 0, 64) == 64000
    assert c.decode_q8_workspace_bytes(1, 8, 2, 96) == 0
    for batch in range(1, 500):
        assert c.decode_q8_workspace_bytes(batch, 8 * batch, batch, 128) == 128000
        assert c.decode_q8_workspace_bytes(batch, 8, 2, 64) == 64000
    assert asked == [64, 96, 128] and len(c._q8_need) == 2


def test_largest_work_list():
    """rows * (max_blocks * block_tokens * head_dim / 4096 + 15) below 2^31,
    with a row for each sequence, KV head and eight query heads of it."""
    lib = _native.lib()
    for batch, qh, kvh, hd, bt, width in ((65535, 64, 8, 64, 16, 1), (60000, 65535, 1, 128, 256, 1),
                                          (1, 128, 1, 128, 128, 1 << 20)):
        rows = batch * kvh * -(-(qh // kvh) // 8)
        units = width * bt * hd // 4096 + 15
        status = decode(lib, batch=batch, qh=qh, kvh=kvh, hd=hd, bt=bt, width=width)
        assert (rows * units < 1 << 31) == (status != 1) or _has_device(lib)
        assert rows * units < 1 << 31 or status == 1


def _has_device(lib):
    """A call that is not refused for its sizes then needs a device (and is
    refused for want of a workspace where there is one)."""
    n = ctypes.c_int(0)
    return lib.mote_cuda_get_device_count(ctypes.byref(n)) == 0 and n.value > 0
