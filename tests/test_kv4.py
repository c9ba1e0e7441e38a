"""CPU tests of the 4-bit KV cache's and the row appends' entry points: argument
checks that need no device."""
from __future__ import annotations

import ctypes as C

import pytest

import qm38


@pytest.fixture()
def none():
    r = qm38.Runtime(-1)
    yield r
    r.close()


P = 1 << 20


def status(call, *args, **kw):
    with pytest.raises(qm38.QmError) as e:
        call(*args, **kw)
    return e.value.status


@pytest.mark.parametrize("shape", [(0, 64, 0, 16), (4, 0, 0, 16), (4, 257, 0, 16), (4, 64, 0, 8)])
def test_cache_shapes(none, shape):
    assert status(none.create_q4_kv_state, *shape) == "QM_ERR_INVALID_ATTENTION_SHAPE"


def test_without_a_device(none):
    assert status(none.create_q4_kv_state, 4, 64) == "QM_ERR_NO_DEVICE"


def test_null_arguments(none):
    lib = qm38.load()
    null = qm38.QM_STATUS.index("QM_ERR_NULL_POINTER")
    h, rows = C.c_void_p(), qm38.KvRows(k=P, v=P)
    seqs, counts = (C.c_void_p * 1)(None), (C.c_uint32 * 1)(1)
    assert lib.qm_kv_create_q4(None, 4, 64, 16, 0, C.byref(h)) == null
    assert lib.qm_kv_create_q4(none.handle, 4, 64, 16, 0, None) == null
    assert lib.qm_kv_bits(None) == 0
    assert lib.qm_kv_read_q4(None, None, None, None, None) == null
    assert lib.qm_kv_append(None, seqs, counts, 1, C.byref(rows)) == null
    assert lib.qm_kv_append(none.handle, None, counts, 1, C.byref(rows)) == null
    assert lib.qm_kv_append(none.handle, seqs, None, 1, C.byref(rows)) == null
    assert lib.qm_kv_append(none.handle, seqs, counts, 1, None) == null
    assert lib.qm_kv_append(none.handle, seqs, counts, 1, C.byref(rows)) == null
    assert lib.qm_kv_append(none.handle, seqs, counts, 1, C.byref(qm38.KvRows(k=P))) == null
    assert lib.qm_kv_load(none.handle, None, 0, 1, P, P) == null
    assert lib.qm_attn_decode_cached(none.handle, seqs, 1, P, None, 4, P) == null
    assert lib.qm_attn_decode_cached(none.handle, None, 1, P, None, 4, P) == null
    assert lib.qm_attn_prefill_cached(none.handle, None, P, None, 4, 1, P) == null


@pytest.mark.parametrize("batch", [0, 65])
def test_batch_sizes(none, batch):
    lib, rows = qm38.load(), qm38.KvRows(k=P, v=P)
    seqs, counts = (C.c_void_p * 65)(), (C.c_uint32 * 65)()
    bad = qm38.QM_STATUS.index("QM_ERR_INVALID_ARGUMENT")
    assert lib.qm_kv_append(none.handle, seqs, counts, batch, C.byref(rows)) == bad
    assert lib.qm_attn_decode_cached(none.handle, seqs, batch, P, None, 4, P) == bad
