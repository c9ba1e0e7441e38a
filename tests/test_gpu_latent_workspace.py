"""GPU tests of the workspaces that latent attention takes from its runtime."""
from __future__ import annotations

import pytest
import torch

from gpu_util import tuned
from test_gpu_latent import FORMS, WIDE, bf16, generator, make_weights

pytestmark = pytest.mark.gpu


def free_bytes():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def test_workspace_does_not_grow_with_every_chunk(torch_dev):
    """A prompt in chunks on a new runtime: what a chunk needs rises with the tokens
    before it (4 MB of keys and values for every 128), and the device's free bytes
    change only as often as that doubles."""
    rank, rope, nope, v = WIDE
    g = generator(71)
    H, rows, chunks = 64, 128, 32
    with tuned(**FORMS["expanded"]) as rt:
        _, _, weights = make_weights(rt, g, H, WIDE)
        cache = rt.create_latent_kv(rank, rope)
        cache.reserve(rows * chunks)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        o = torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev)
        before, seen = free_bytes(), []
        for _ in range(chunks):
            rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
            seen.append(free_bytes())
        if before - seen[-1] < 64 << 20:
            pytest.skip(f"free-memory reading did not see the workspace ({before - seen[-1]} B)")
        # From one chunk's to 32 chunks': the first allocation and five doublings,
        # and one more where the first is just short of a power of two.
        changes = sum(a != b for a, b in zip([before, *seen], seen))
        assert changes <= 7, f"{changes} changes of the workspace in {chunks} chunks"
        weights.close()
        cache.close()


def test_partial_sums_do_not_grow_with_every_step(torch_dev):
    """The same of the partial sums, which rise with the splits of a longer cache."""
    rank, rope, nope, v = WIDE
    g = generator(72)
    H, step = 128, 512
    with tuned() as rt:
        _, _, weights = make_weights(rt, g, H, WIDE)
        cache = rt.create_latent_kv(rank, rope)
        cache.reserve(32768)
        kv = bf16(g, step, rank + rope)
        q, one = bf16(g, 1, H, nope + rope), bf16(g, 1, rank + rope)
        o = torch.empty(1, H, v, dtype=torch.bfloat16, device=torch_dev)
        before, seen = free_bytes(), []
        for _ in range(40):
            cache.append(kv, None, 0.0, step - 1)
            rt.latent_attention(weights, [cache], q, one, None, 0.0, o)
            seen.append(free_bytes())
        if before - seen[-1] < 16 << 20:
            pytest.skip(f"free-memory reading did not see the partial sums ({before - seen[-1]} B)")
        # 1 MB to 34 MB at most: six doublings, one of them with the first scratch.
        changes = sum(a != b for a, b in zip([before, *seen], seen))
        assert changes <= 7, f"{changes} changes of the workspace in 40 steps"
        weights.close()
        cache.close()
