"""GPU tests of decode attention over 4-bit caches within its own rounding bound, and over
values that differ widely."""
from __future__ import annotations

import pytest
import torch

from kv4_tight import beyond, decode_bound
from kv4_util import attention, check, read, values
from test_gpu_kv4 import DEV, bf16, generator, make, randn

pytestmark = pytest.mark.gpu

SHAPES = [(8, 2, 64), (64, 8, 128), (24, 4, 256), (20, 5, 80), (16, 1, 128), (13, 1, 256), (4, 2, 37)]


@pytest.mark.parametrize("n", [1, 2, 5, 16, 17, 31, 32])
@pytest.mark.parametrize("H,KVH,D", SHAPES)
def test_decode_weights(rt, H, KVH, D, n):
    """Appending and of cached tokens, and as rows of a prompt."""
    g = generator(100 + n)
    cache = make(rt, 4, KVH, D)
    if n > 1:
        rt.kv_append([cache], [n - 1], bf16(g, n - 1, KVH, D), bf16(g, n - 1, KVH, D))
    q, k, v = bf16(g, n, H, D, std=0.01), randn(g, 1, KVH, D), randn(g, 1, KVH, D)
    o = torch.empty_like(q)
    rt.gqa_attention_q8([cache], q[-1:], None, k, v, H, o[-1:])
    parts = read(cache)
    want, bound = decode_bound(q[-1:], *parts, n - 1)
    assert beyond(o[-1:], want, bound) == 0
    o.fill_(7.0)
    rt.gqa_attention([cache], q[-1:], None, H, o[-1:])
    assert beyond(o[-1:], want, bound) == 0
    o.fill_(7.0)
    rt.gqa_attention_prefill(cache, q, None, H, n, o)
    assert beyond(o, *decode_bound(q, *parts, 0)) == 0
    cache.close()


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("power", [-60, 9, 40, 90])
@pytest.mark.parametrize("H,KVH,D", [(8, 1, 128), (12, 2, 256), (8, 2, 64), (40, 4, 256)])
def test_few_rows_over_one_far_group(rt, H, KVH, D, power, rows):
    """A token whose first 64 values are far larger or smaller: the other groups keep theirs."""
    g = generator(101)
    n = 900
    cache = make(rt, 4, KVH, D)
    k, v = bf16(g, n, KVH, D, std=0.2), bf16(g, n, KVH, D)
    v[40, :, :64] *= 2.0 ** power
    rt.kv_append([cache], [n], k, v)
    q = bf16(g, rows, H, D)
    o = torch.empty_like(q)
    want, bound = attention(q, None, values(cache), n - rows)
    rt.gqa_attention_prefill(cache, q, None, H, rows, o)
    check(o, want, bound)
    rt.gqa_attention([cache], q[-1:].contiguous(), None, H, o[:1])
    check(o[:1], want[-1:], bound[-1:])
    cache.close()
