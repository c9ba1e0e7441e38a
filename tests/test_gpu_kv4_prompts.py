"""GPU tests of prompts over 4-bit caches where something that they usually have is not
there, and of values that differ widely."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import qm38
from kv4_util import attention, check, values
from test_gpu_kv4 import DEV, bf16, fill, generator, make, randn

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# No room for the partials of splits
# ---------------------------------------------------------------------------
# Prompts whose plan splits blocks of columns, a few rows that go as a decode step, and
# one that is not split.
WITHOUT = [(20, 5, 80, 333, 0), (64, 8, 128, 513, 0), (24, 4, 256, 512, 13), (24, 4, 256, 1000, 0), (3, 1, 256, 700, 0),
           (32, 8, 64, 1101, 0), (16, 2, 64, 300, 4000), (24, 4, 256, 5, 3001), (16, 2, 128, 100, 0)]


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("H,KVH,D,rows,cached", WITHOUT)
def test_prompts_on_the_per_thread_stream(rt, H, KVH, D, rows, cached, gated):
    """Nothing may grow on that stream: a prompt goes without splits."""
    g = generator(60 + rows)
    cache, usual = make(rt, 4, KVH, D), make(rt, 4, KVH, D)
    if cached:
        fill(rt, cache, generator(3), cached)
        fill(rt, usual, generator(3), cached)
    cache.reserve(rows)
    q, k, v = bf16(g, rows, H, D, std=1.5), randn(g, rows, KVH, D), randn(g, rows, KVH, D)
    gate = bf16(g, rows, H, D) if gated else None
    o, o_usual = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV), torch.empty_like(q)
    rt.gqa_attention_q8_prefill(usual, q, gate, k, v, H, rows, o_usual)
    torch.cuda.synchronize()
    own = qm38.Runtime(0)
    try:
        assert own.lib.qm_runtime_set_stream(own.handle, C.c_void_p(2)) == 0
        own.gqa_attention_q8_prefill(cache, q, gate, k, v, H, rows, o)
        torch.cuda.synchronize()
    finally:
        own.set_stream(None)
        own.close()
    want, bound = attention(q, gate, values(cache), cached)
    check(o, want, bound)
    check(o_usual, want, bound)
    cache.close()
    usual.close()


@pytest.mark.parametrize("H,KVH,D,rows,cached", WITHOUT)
def test_captured_prompts(rt, H, KVH, D, rows, cached):
    """The same under capture, and every replay of the graph."""
    g = generator(70 + rows)
    cache = make(rt, 4, KVH, D)
    if cached:
        fill(rt, cache, g, cached)
    cache.reserve(rows)
    q, k, v = bf16(g, rows, H, D, std=1.5), randn(g, rows, KVH, D), randn(g, rows, KVH, D)
    gate = bf16(g, rows, H, D)
    o = torch.empty_like(q)
    torch.cuda.synchronize()
    own, stream, graph = qm38.Runtime(0), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            own.set_stream(stream)
            own.gqa_attention_q8_prefill(cache, q, gate, k, v, H, rows, o)
        first = None
        for step in range(3):
            o.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            if first is None:
                first = o.clone()
                check(o, *attention(q, gate, values(cache), cached))
            assert torch.equal(o, first)
            q_other = bf16(g, rows, H, D)  # (eager work between)
            again = torch.empty_like(o)
            rt.gqa_attention_prefill(cache, q_other, None, H, rows, again)
        check(again, *attention(q_other, None, values(cache), cached))
    finally:
        own.set_stream(None)
        own.close()
        cache.close()
