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


# ---------------------------------------------------------------------------
# Values that differ widely between groups and tiles
# ---------------------------------------------------------------------------
def over(rt, k, v, H, rows, std=1.0, gated=False):
    """A prompt's last rows over cached bf16 rows, checked against the formula."""
    n, KVH, D = k.shape
    g = generator(81)
    cache = make(rt, 4, KVH, D)
    rt.kv_append([cache], [n], k, v)
    q = bf16(g, rows, H, D, std=std)
    gate = bf16(g, rows, H, D) if gated else None
    o = torch.empty_like(q)
    rt.gqa_attention_prefill(cache, q, gate, H, rows, o)
    kv = values(cache)
    cache.close()
    check(o, *attention(q, gate, kv, n - rows))


SPREAD = [(8, 1, 128), (12, 2, 256), (8, 2, 64), (8, 2, 100), (40, 4, 256)]


@pytest.mark.parametrize("token", [3, 40, 700])
@pytest.mark.parametrize("power", [-60, -20, 9, 40, 90])
@pytest.mark.parametrize("H,KVH,D", SPREAD)
def test_one_group_of_one_token(rt, H, KVH, D, power, token):
    """A token whose first 64 values are far larger (or smaller) than all others: the other
    groups and tokens keep theirs."""
    g = generator(80)
    k, v = bf16(g, 900, KVH, D, std=0.2), bf16(g, 900, KVH, D)
    v[token, :, :64] *= 2.0 ** power
    over(rt, k, v, H, 130, gated=power == 40)


@pytest.mark.parametrize("std", [0.2, 4.0])
@pytest.mark.parametrize("H,KVH,D", SPREAD)
def test_groups_that_cross(rt, H, KVH, D, std):
    """Groups that grow and shrink against one another over the tiles, by 2^5 a tile and up to
    2^50 in all, with weights spread or on single tokens."""
    g = generator(82)
    n, tile = 640, torch.arange(640, device=DEV) // 32
    v = randn(g, n, KVH, D)
    for i, at in enumerate(range(0, D, 64)):
        power = (5.0 * tile if i % 2 == 0 else 50.0 - 5.0 * tile).clamp(0, 50)
        v[..., at:at + 64] *= (2.0 ** power)[:, None, None]
    over(rt, bf16(g, n, KVH, D), v.to(torch.bfloat16), H, 200, std=std)


@pytest.mark.parametrize("H,KVH,D", SPREAD)
def test_tiles_of_zeros(rt, H, KVH, D):
    """Tokens of zeros before, between and behind others, in some groups or all."""
    g = generator(83)
    k, v = bf16(g, 500, KVH, D), bf16(g, 500, KVH, D)
    v[:96] = 0
    v[200:300, :, :64] = 0
    v[300:364] *= 2.0 ** -30
    v[480:] = 0
    over(rt, k, v, H, 200)


@pytest.mark.parametrize("H,KVH,D", SPREAD)
def test_large_values_of_small_weight(rt, H, KVH, D):
    """Values 2^40 larger whose weights are about 2^-40: their part counts as others' do."""
    g = generator(84)
    n = 512
    k, v = torch.zeros(n, KVH, D, device=DEV), randn(g, n, KVH, D)
    k[..., 0] = 1.0
    far = torch.zeros(n, dtype=torch.bool, device=DEV)
    far[64:96] = far[300:320] = True
    k[far, :, 0] = -1.0
    v[far] *= 2.0 ** 40
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    cache = make(rt, 4, KVH, D)
    rt.kv_append([cache], [n], k, v)
    # Scores of +-s / sqrt(D): weights 2^-40 apart.
    s = 20 * 0.6931471805599453 * D ** 0.5
    q = torch.zeros(130, H, D, device=DEV)
    q[..., 0] = s
    q = (q + 0.1 * randn(g, *q.shape)).to(torch.bfloat16)
    o = torch.empty_like(q)
    rt.gqa_attention_prefill(cache, q, None, H, 130, o)
    check(o, *attention(q, None, values(cache), n - 130))
    cache.close()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [-18, -16, -15, -14, -13, -12, -10, -8, 3, 4, 4.5, 5, 6, 7, 7.5, 8, 8.5, 9])
def test_sizes_around_what_one_unit_takes(rt, D, power):
    """Later tokens smaller or larger than the first tile's by a few powers of two, their values
    all on one side of zero, as far from their group's middle as codes go."""
    g = generator(85)
    n = 300
    k, v = bf16(g, n, 2, D, std=0.3), randn(g, n, 2, D)
    v[100:] = -1.0 - 15.0 * torch.randint(0, 16, v[100:].shape, generator=g, device=DEV) / 15.0
    v[100:] *= 2.0 ** power / 8
    over(rt, k, v.to(torch.bfloat16), 16, 140)


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("H,KVH,D,rows", [(64, 8, 128, 513), (24, 4, 256, 700), (20, 5, 80, 333), (3, 1, 256, 1101),
                                          (32, 8, 64, 700), (6, 2, 37, 513)])
def test_far_sizes_in_split_prompts(rt, H, KVH, D, rows, gated):
    """Some workgroups of a split prompt meet the large token, others do not; rows that are no
    multiple of a workgroup's."""
    g = generator(86)
    cache = make(rt, 4, KVH, D)
    q, k, v = bf16(g, rows, H, D), randn(g, rows, KVH, D, std=0.3), randn(g, rows, KVH, D)
    v[rows // 2, :, :min(D, 64)] *= 2.0 ** 30
    gate = bf16(g, rows, H, D) if gated else None
    o = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    rt.gqa_attention_q8_prefill(cache, q, gate, k, v, H, rows, o)
    check(o, *attention(q, gate, values(cache), 0))
    cache.close()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("H,KVH,D", [(8, 2, 64), (8, 2, 128), (12, 2, 256), (20, 4, 100)])
def test_nan_beside_far_sizes(rt, H, KVH, D, kind):
    """A NaN, tokens that were dropped and a size far from the others."""
    g = generator(87)
    cache = make(rt, 4, KVH, D)
    x = [bf16(g, 260, KVH, D, std=0.5) for _ in range(2)]
    x[kind][130, 1, D - 3] = float("nan")
    x[1][40] *= 2.0 ** 25
    rt.kv_append([cache], [260], *x)
    bad = torch.full((40, KVH, D), float("inf"), dtype=torch.bfloat16, device=DEV)
    rt.kv_append([cache], [40], bad, bad)
    cache.truncate(260)
    rows, per = 200, H // KVH
    q = bf16(g, rows, H, D)
    o = torch.empty_like(q)
    rt.gqa_attention_prefill(cache, q, None, H, rows, o)  # row i is token 60 + i
    nan = torch.zeros(rows, H, D, dtype=torch.bool, device=DEV)
    nan[70:, per:2 * per, (D - 3) // 64 * 64 if kind else 0:] = True
    assert torch.equal(torch.isnan(o), nan)
    clean = [(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in values(cache)]
    want, bound = attention(q, None, clean, 60)
    check(o.masked_fill(nan, 0.0), want.masked_fill(nan, 0.0), bound)
    cache.close()
