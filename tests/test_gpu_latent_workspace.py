"""GPU tests of the workspaces that latent attention takes from its runtime."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import qm38
from gpu_util import to_dev, tuned
from qm38 import synth
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


def _q4(torch_dev, rng, n, k):
    mat = tuple(to_dev(a, torch_dev) for a in synth.q4_matrix(rng, n, k))
    return mat, qm38.Runtime.job(*mat, n)


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_a_graph_keeps_the_workspaces_that_latent_attention_outgrows(torch_dev, form):
    """Captured projections hold the addresses of the runtime's workspaces (the MLP's
    inner rows, split sums, converted activations).  An eager prompt that needs larger
    ones leaves those to the graph: every replay gives the eager call's bits."""
    rank, rope, nope, v = WIDE
    g, rng = generator(73), np.random.default_rng(73)
    E, F, H, rows = 512, 1024, 64, 512
    with tuned(**FORMS[form]) as rt:
        _, _, weights = make_weights(rt, g, H, WIDE)
        (m0, gate), (m1, up), (m2, down) = _q4(torch_dev, rng, F, E), _q4(torch_dev, rng, F, E), _q4(torch_dev, rng, E, F)
        x = [bf16(g, n, E, std=0.3) for n in (1, 40)]
        eager, got = ([torch.zeros(len(a), E, dtype=torch.bfloat16, device=torch_dev) for a in x] for _ in range(2))

        def mlp(outs):
            for a, y in zip(x, outs):
                rt.q4_mlp(gate, up, down, a, E, len(a), y)

        mlp(eager)  # sizes the workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            rt.set_stream(torch.cuda.current_stream())
            mlp(got)
        rt.set_stream(torch.cuda.current_stream())
        cache = rt.create_latent_kv(rank, rope)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        o = torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev)
        for _ in range(4):
            rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
            taken = torch.full((1 << 22,), float("nan"), device=torch_dev)  # of what has been freed, if anything has
            for a, y in zip(x, got):
                a.copy_(bf16(g, len(a), E, std=0.3))
                y.zero_()
            mlp(eager)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(eager, got):
                assert torch.isfinite(a).all() and torch.equal(a, b)
            assert torch.isnan(taken).all()
        del graph
        weights.close()
        cache.close()


def test_a_large_workspace_is_not_doubled(torch_dev):
    """Above 2 GB a workspace is what the call needs, rounded up to a GB."""
    rank, rope, nope, v = WIDE
    g = generator(74)
    H, rows, cached = 64, 2048, 80000
    with tuned(QM38_LATENT_FORM=2, QM38_LATENT_MB=8192) as rt:
        _, _, weights = make_weights(rt, g, H, WIDE)
        cache = rt.create_latent_kv(rank, rope)
        cache.reserve(cached + rows)
        cache.append(bf16(g, cached, rank + rope), None, 0.0, cached)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        o = torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev)
        before = free_bytes()
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
        taken = before - free_bytes()
        if taken == 0:
            pytest.skip("free-memory reading did not see the workspace")
        # Keys and values of 64 heads, 512 bytes a token each, and the unpacked cache.
        need = (cached + rows) * (64 * 512 + 1024 + 128 + 8)
        assert need <= taken <= need + (1 << 30) + (64 << 20)
        weights.close()
        cache.close()
