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


# ---------------------------------------------------------------------------
# Tensors that the Python calls cannot pass on as rows
# ---------------------------------------------------------------------------
class Sequence:
    """A cache's place in an argument list, which no check of these dereferences."""
    handle, kv_heads, head_dim = None, 2, 64


def rows(n, heads=2, dtype=None):
    import torch
    return torch.zeros(n, heads, 64, dtype=dtype or torch.bfloat16)


def not_rows():
    import torch
    return {
        "one row for all": rows(1).expand(5, 2, 64),
        "heads before rows": torch.zeros(2, 5, 64, dtype=torch.bfloat16).transpose(0, 1),
        "every other element": torch.zeros(5, 2, 128, dtype=torch.bfloat16)[..., ::2],
        "one head for all": torch.zeros(5, 1, 64, dtype=torch.bfloat16).expand(5, 2, 64),
        "fp32": rows(5, dtype=torch.float32),
        "fp16": rows(5, dtype=torch.float16),
    }


@pytest.mark.parametrize("what", sorted(not_rows()))
@pytest.mark.parametrize("name", ["k", "v", "q", "q_out"])
def test_appended_tensors(none, name, what):
    tensors = dict(k=rows(5), v=rows(5), q=rows(5), q_out=rows(5))
    tensors[name] = not_rows()[what]
    turn = qm38.RotaryConfig(64, False, 1e4)
    with pytest.raises(ValueError, match=f"^{name}:"):
        none.kv_append([Sequence()], [5], tensors["k"], tensors["v"], rotary=turn, q=tensors["q"],
                       q_out=tensors["q_out"], num_heads=2)


@pytest.mark.parametrize("how", ["int64", "float32", "strided", "expanded"])
def test_appended_positions(none, how):
    import torch
    bad = {"int64": torch.arange(5), "float32": torch.zeros(5), "strided": torch.zeros(10, dtype=torch.int32)[::2],
           "expanded": torch.zeros(1, dtype=torch.int32).expand(5)}[how]
    with pytest.raises(ValueError, match="^positions:"):
        none.kv_append([Sequence()], [5], rows(5), rows(5), rotary=qm38.RotaryConfig(64, False, 1e4), positions=bad)


def test_counts_of_other_sequences(none):
    for counts in ([5], [2, 2, 1], []):
        with pytest.raises(ValueError, match="counts"):
            none.kv_append([Sequence(), Sequence()], counts, rows(5), rows(5))


def test_rows_that_are_taken(none):
    """Rows any stride apart, raw addresses and integers of 16 bits reach the library."""
    import torch
    fused = torch.zeros(5, 3 * 2 * 64, dtype=torch.bfloat16)
    q, k, v = fused.split(2 * 64, 1)
    turn = qm38.RotaryConfig(64, False, 1e4)
    for args, kw in [((k, v), dict(rotary=turn, q=q, q_out=q, num_heads=2)),
                     ((k.unflatten(1, (2, 64)), v.unflatten(1, (2, 64))), {}),
                     ((k[:1], rows(1).expand(1, 2, 64)), {}),
                     ((rows(5, dtype=torch.int16), P), dict(positions=torch.zeros(5, dtype=torch.int32), rotary=turn))]:
        assert status(none.kv_append, [Sequence()], [len(args[0])], *args, **kw) == "QM_ERR_NULL_POINTER"


@pytest.mark.parametrize("what", sorted(set(not_rows()) | {"too few"}))
@pytest.mark.parametrize("part", [0, 1])
def test_loaded_tensors(none, part, what):
    cache = qm38.KvCache(none, 2, 64, 16, 0, handle=C.c_void_p(None))
    out = [rows(5), rows(5)]
    out[part] = rows(4) if what == "too few" else not_rows()[what]
    with pytest.raises(ValueError, match="^" + "kv"[part] + ":"):
        cache.load(0, 5, *out)
    assert status(cache.load, 0, 5, rows(5), P) == "QM_ERR_NULL_POINTER"
    assert status(cache.load, 0, 5, None, rows(7)) == "QM_ERR_NULL_POINTER"


@pytest.mark.parametrize("what", sorted(not_rows()))
@pytest.mark.parametrize("name", ["q", "gate", "o"])
def test_attended_tensors(none, name, what):
    tensors = dict(q=rows(5), gate=rows(5), o=rows(5))
    tensors[name] = not_rows()[what]
    with pytest.raises(ValueError, match=f"^{name}:"):
        none.gqa_attention([Sequence()] * 5, tensors["q"], tensors["gate"], 2, tensors["o"])
    with pytest.raises(ValueError, match=f"^{name}:"):
        none.gqa_attention_prefill(Sequence(), tensors["q"], tensors["gate"], 2, 5, tensors["o"])
