"""CPU tests of the latent attention and rotary entry points: argument checks on
a runtime without a device, which never touches a GPU."""
from __future__ import annotations

import ctypes as C

import pytest

import qm38


@pytest.fixture()
def none():
    r = qm38.Runtime(-1)
    yield r
    r.close()


P = 1 << 20  # addresses that only the checks look at
Q = 1 << 30


def status(call, *args, **kw):
    with pytest.raises(qm38.QmError) as e:
        call(*args, **kw)
    return e.value.status


@pytest.mark.parametrize("want,config,tensors,rows,kw", [
    ("QM_ERR_NO_DEVICE", dict(rotary_dim=64), [(P, Q, 4, 192, 128)], 3, {}),
    ("QM_ERR_NO_DEVICE", dict(rotary_dim=64), [(P, P, 4, 192, 128)], 3, {}),
    ("QM_ERR_NO_DEVICE", dict(rotary_dim=64, scaling="yarn", factor=2.0, original_positions=10), [(P, Q, 1, 64, 0)], 1, {}),
    # Columns of one buffer, row by row: no element is shared.
    ("QM_ERR_NO_DEVICE", dict(rotary_dim=64), [(P, P + 128, 1, 64, 0, 128, 128)], 9, {}),
    ("QM_ERR_NO_DEVICE", dict(rotary_dim=64), [(P + 128, P, 1, 64, 0, 128, 128)], 9, {}),
    ("QM_ERR_NO_DEVICE", dict(rotary_dim=64), [(P, P, 1, 64, 0, 640, 640), (P + 128, P + 128, 1, 576, 512, 640, 640)], 9, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [(P, P + 126, 1, 64, 0, 128, 128)], 9, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [(P + 126, P, 1, 64, 0, 128, 128)], 9, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [(P, P, 1, 64, 0, 64, 128)], 9, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [(P, P + 64, 4, 192, 128)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [(P, Q, 1, 64, 0), (P, Q, 1, 64, 0)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [(P, Q, 1, 64, 0), (Q, Q + 4096, 1, 64, 0)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [(P + 4096 * i, Q + 4096 * i, 1, 64, 0) for i in range(5)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64), [(P, Q, 4, 192, 0, 100, 0)], 3, {}),
    ("QM_ERR_EMPTY_DIMENSION", dict(rotary_dim=64), [(P, Q, 4, 192, 128)], 0, {}),
    ("QM_ERR_EMPTY_DIMENSION", dict(rotary_dim=64), [(P, Q, 0, 192, 128)], 3, {}),
    ("QM_ERR_INVALID_ATTENTION_SHAPE", dict(rotary_dim=64), [(P, Q, 4, 192, 129)], 3, {}),
    ("QM_ERR_INVALID_ATTENTION_SHAPE", dict(rotary_dim=63), [(P, Q, 4, 192, 0)], 3, {}),
    ("QM_ERR_INVALID_ATTENTION_SHAPE", dict(rotary_dim=258), [(P, Q, 4, 512, 0)], 3, {}),
    ("QM_ERR_INVALID_ATTENTION_SHAPE", dict(rotary_dim=0), [(P, Q, 4, 512, 0)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64, theta=1.0), [(P, Q, 1, 64, 0)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64, theta=float("nan")), [(P, Q, 1, 64, 0)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64, scaling="linear", factor=0.5), [(P, Q, 1, 64, 0)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64, scaling="yarn", factor=2.0), [(P, Q, 1, 64, 0)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64, scaling="yarn", factor=2.0, original_positions=9, beta_fast=1.0),
     [(P, Q, 1, 64, 0)], 3, {}),
    ("QM_ERR_INVALID_ARGUMENT", dict(rotary_dim=64, attention_factor=-1.0), [(P, Q, 1, 64, 0)], 3, {}),
    ("QM_ERR_DIMENSION_OVERFLOW", dict(rotary_dim=64), [(P, Q, 1, 64, 0)], 3, dict(position_base=2 ** 32 - 2)),
    ("QM_ERR_DIMENSION_OVERFLOW", dict(rotary_dim=64), [(P, Q, 2 ** 25, 64, 0)], 3, {}),
    ("QM_ERR_DIMENSION_OVERFLOW", dict(rotary_dim=64), [(P, Q, 1, 64, 0, 2 ** 61, 0)], 3, {}),
    ("QM_ERR_MISALIGNED", dict(rotary_dim=64), [(P + 1, Q, 1, 64, 0)], 3, {}),
    ("QM_ERR_MISALIGNED", dict(rotary_dim=64), [(P, Q, 1, 64, 0)], 3, dict(positions=P + 2)),
    ("QM_ERR_NULL_POINTER", dict(rotary_dim=64), [(P, None, 1, 64, 0)], 3, {}),
])
def test_rotary_arguments(none, want, config, tensors, rows, kw):
    assert status(none.rotary, qm38.RotaryConfig(**config), tensors, rows, **kw) == want


def test_unknown_layout_and_scaling(none):
    c = qm38.RotaryConfig(64)
    c.layout = 2
    assert status(none.rotary, c, [(P, Q, 1, 64, 0)], 1) == "QM_ERR_INVALID_ARGUMENT"
    c.layout, c.scaling = 0, 3
    assert status(none.rotary, c, [(P, Q, 1, 64, 0)], 1) == "QM_ERR_INVALID_ARGUMENT"


@pytest.mark.parametrize("rank,rope", [(0, 64), (520, 64), (12, 64), (512, 0), (512, 72), (512, 4)])
def test_cache_shapes(none, rank, rope):
    assert status(none.create_latent_kv, rank, rope) == "QM_ERR_INVALID_ATTENTION_SHAPE"


def test_without_a_device(none):
    assert status(none.create_latent_kv, 512, 64) == "QM_ERR_NO_DEVICE"
    cfg = qm38.LatentConfig(4, 512, 128, 64, 128, 0.1)
    assert status(none.create_latent_weights, cfg, P) == "QM_ERR_NO_DEVICE"
    assert status(none.create_latent_weights, cfg, qm38.Q4Job(P, P, P, 4 * 256)) == "QM_ERR_NO_DEVICE"
    assert status(none.create_latent_weights, cfg, qm38.Q4Job(P, P + 4, P, 4 * 256)) == "QM_ERR_MISALIGNED"
    assert status(none.create_latent_weights, cfg, qm38.Q4Job(P, None, P, 4 * 256)) == "QM_ERR_NULL_POINTER"
    assert status(none.create_latent_weights, cfg, None) == "QM_ERR_NULL_POINTER"


def test_null_arguments(none):
    lib = qm38.load()
    null = qm38.QM_STATUS.index("QM_ERR_NULL_POINTER")
    cfg, h = qm38.LatentConfig(4, 512, 128, 64, 128, 0.1), C.c_void_p()
    assert lib.qm_rotary(none.handle, None, None, 1, 1, None, 0) == null
    assert lib.qm_latent_kv_create(None, 512, 64, 0, C.byref(h)) == null
    assert lib.qm_latent_kv_create(none.handle, 512, 64, 0, None) == null
    assert lib.qm_latent_kv_clone(None, C.byref(h)) == null
    assert lib.qm_latent_kv_reserve(None, 1) == null
    assert lib.qm_latent_kv_truncate(None, 0) == null
    assert lib.qm_latent_kv_read(None, None, None) == null
    assert lib.qm_latent_append(none.handle, None, P, None, 0.0, 1) == null
    assert lib.qm_latent_load(none.handle, None, 0, 1, P) == null
    assert lib.qm_latent_weights_create(none.handle, C.byref(cfg), P, None) == null
    assert lib.qm_latent_decode(none.handle, None, None, 1, P, P, None, 0.0, P) == null
    assert lib.qm_latent_prefill(none.handle, None, None, P, P, None, 0.0, 1, P) == null
    assert lib.qm_latent_kv_length(None) == lib.qm_latent_kv_capacity(None) == 0
    lib.qm_latent_kv_destroy(None)
    lib.qm_latent_weights_destroy(None)
