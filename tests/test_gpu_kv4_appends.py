"""GPU tests of qm_kv_append: memory that queries must not be written over."""
from __future__ import annotations

import pytest
import torch

import qm38
from test_gpu_kv4 import DEV, bf16, generator, make

pytestmark = pytest.mark.gpu


def test_queries_over_the_positions(rt):
    """q_out may lie on no input: not on the positions that keys are rotated by either."""
    g = generator(90)
    H, KVH, D, n = 4, 2, 64, 8
    cache = make(rt, 4, KVH, D)
    k, v, q = (bf16(g, n, heads, D) for heads in (KVH, KVH, H))
    turn = qm38.RotaryConfig(64, False, 1e4)
    memory = torch.full((n * H * D + 2 * n,), 2.0, dtype=torch.bfloat16, device=DEV)
    out = memory[:n * H * D].view(n, H, D)
    last = memory.view(torch.int32)
    for at in (0, 5, n * H * D // 2 - 1):  # positions that begin in the output
        with pytest.raises(qm38.QmError) as e:
            rt.kv_append([cache], [n], k, v, rotary=turn, positions=last[at:at + n], q=q, q_out=out, num_heads=H)
        assert e.value.status == "QM_ERR_INVALID_ARGUMENT"
    # ... or end in it.
    with pytest.raises(qm38.QmError) as e:
        rt.kv_append([cache], [n], k, v, rotary=turn, positions=last[:n], q=q,
                     q_out=memory[2 * n - 2:2 * n - 2 + n * H * D].view(n, H, D), num_heads=H)
    assert e.value.status == "QM_ERR_INVALID_ARGUMENT"
    torch.cuda.synchronize()
    assert (memory == 2).all() and cache.sequence_length == 0
    # Right behind it they are fine.
    positions = last[n * H * D // 2:]
    positions.copy_(torch.arange(n, dtype=torch.int32, device=DEV) + 7)
    rt.kv_append([cache], [n], k, v, rotary=turn, positions=positions, q=q, q_out=out, num_heads=H)
    want = torch.empty_like(q)
    rt.rotary(turn, [(q, want, H, D, 0)], n, position_base=7)
    assert torch.equal(out, want) and torch.equal(positions.cpu(), torch.arange(n, dtype=torch.int32) + 7)
    cache.close()
