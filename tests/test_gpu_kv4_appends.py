"""GPU tests of qm_kv_append: memory that queries must not be written over, and the bits
of their rotation whatever the rows' alignment."""
from __future__ import annotations

import numpy as np
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


@pytest.mark.parametrize("shift,extra", [(0, 0), (0, 24), (1, 0), (4, 8), (0, 3), (1, 5), (8, 1)])
@pytest.mark.parametrize("D,rd,interleaved", [(128, 128, False), (128, 64, True), (256, 256, False), (80, 48, True)])
def test_query_bits_of_any_alignment(rt, D, rd, interleaved, shift, extra):
    """Queries have the bits that qm_rotary gives for the same rows at the same place."""
    g = generator(91)
    H, KVH, n = 5, 1, 37
    cache = make(rt, 4, KVH, D)
    width = H * D + extra
    rows = bf16(g, n * width + shift)[shift:].view(n, width)
    q, k = rows[:, :H * D], bf16(g, n, KVH, D)
    turn = qm38.RotaryConfig(rd, interleaved, 1e4)
    buffer = torch.zeros(n * width + shift, dtype=torch.bfloat16, device=DEV)
    got, want = (buffer.clone()[shift:].view(n, width) for _ in range(2))
    rt.kv_append([cache], [n], k, k, rotary=turn, q=q, q_out=got[:, :H * D], num_heads=H)
    rt.rotary(turn, [(q, want[:, :H * D], H, D, 0, width, width)], n)
    assert torch.equal(got, want)
    assert np.isfinite(got.float().cpu().numpy()).all() and not (got[:, H * D:] != 0).any()
    cache.close()
