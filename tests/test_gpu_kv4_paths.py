"""GPU tests of the 4-bit KV cache along the paths that callers take: prompts, steps
and batches together, long calls, several runtimes and streams, decode layers, and the
calls that are refused."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

import qm38
from kv4_util import attention, check, frequencies, read, rotated, values
from test_gpu_decode import EPS, FULL, Model, _hidden, _hidden0, _manual_token, _positions, _state_with
from test_gpu_kv4 import DEV, SHAPES, bf16, fill, generator, make, near_rows, randn, same_rows

pytestmark = pytest.mark.gpu


def equal(a, b):
    """Two caches' content, bit for bit."""
    assert a.sequence_length == b.sequence_length
    assert all(np.array_equal(x, y) for x, y in zip(a.read(), b.read()))


# ---------------------------------------------------------------------------
# Prefill beyond the few rows that go as a decode step
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows,cached", [(65, 0), (130, 47), (257, 31), (40, 5001), (9, 20001)])
@pytest.mark.parametrize("shape", SHAPES)
def test_prefill_of_many_rows(rt, shape, rows, cached):
    g = generator(sum(shape) + rows)
    H, KVH, D = shape
    cache = make(rt, 4, KVH, D)
    if cached:
        fill(rt, cache, g, cached)
    q, k, v = bf16(g, rows, H, D, std=1.5), randn(g, rows, KVH, D), randn(g, rows, KVH, D)
    gate = bf16(g, rows, H, D) if rows % 2 else None
    o = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    rt.gqa_attention_q8_prefill(cache, q, gate, k, v, H, rows, o)
    want, bound = attention(q, gate, values(cache), cached)
    check(o, want, bound)
    again = torch.empty_like(o)
    rt.gqa_attention_prefill(cache, q, gate, H, rows, again)
    assert torch.equal(again, o)
    # One row as a decode step.
    cache.truncate(cached + rows - 1)
    one = torch.empty_like(o[:1])
    rt.gqa_attention_q8([cache], q[-1:], gate[-1:] if gate is not None else None, k[-1:], v[-1:], H, one)
    check(one, want[-1:], bound[-1:])
    cache.close()


@pytest.mark.parametrize("rows,cached", [(513, 0), (700, 13), (1101, 0)])
@pytest.mark.parametrize("shape", [(64, 8, 128), (20, 5, 80), (24, 4, 256), (32, 8, 64), (16, 1, 128), (6, 2, 37)])
def test_prompts_split_by_blocks(rt, shape, rows, cached):
    """Blocks of columns with different numbers of workgroups, gated (odd rows) and not."""
    test_prefill_of_many_rows(rt, shape, rows, cached)


@pytest.mark.parametrize("rows", [2100, 2101])
@pytest.mark.parametrize("shape", [(2, 1, 64), (3, 1, 256)])
def test_prompts_in_many_splits(rt, shape, rows):
    test_prefill_of_many_rows(rt, shape, rows, 0)


@pytest.mark.parametrize("shape", [(8, 2, 64), (8, 2, 128), (12, 2, 256), (40, 2, 256)])
@pytest.mark.parametrize("kind", [0, 1])
def test_nan_reaches_many_rows(rt, kind, shape):
    """A NaN among many tiles, and tokens that were dropped."""
    g = generator(20 + kind)
    H, KVH, D = shape
    if H // KVH > 16:
        KVH = 4
    cache = make(rt, 4, KVH, D)
    x = [bf16(g, 260, KVH, D) for _ in range(2)]
    x[kind][130, 1, D - 3] = math.nan
    rt.kv_append([cache], [260], *x)
    bad = torch.full((40, KVH, D), math.inf, dtype=torch.bfloat16, device=DEV)
    rt.kv_append([cache], [40], bad, bad)
    cache.truncate(260)
    rows = 200
    q = bf16(g, rows, H, D)
    o = torch.empty_like(q)
    rt.gqa_attention_prefill(cache, q, None, H, rows, o)  # row i is token 60 + i
    per = H // KVH
    nan = torch.zeros(rows, H, D, dtype=torch.bool, device=DEV)
    nan[70:, per:2 * per, (D - 3) // 64 * 64 if kind else 0:] = True
    assert torch.equal(torch.isnan(o), nan)
    clean = values(cache)
    clean = [(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in clean]
    want, bound = attention(q, None, clean, 60)
    check(o.masked_fill(nan, 0.0), want.masked_fill(nan, 0.0), bound)
    cache.close()


@pytest.mark.parametrize("std_k,std_v", [(1e-12, 1e-12), (1.0, 1e20), (1e4, 1.0), (1.0, 1e-30), (1e-3, 1e36)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_magnitudes_of_many_rows(rt, D, std_k, std_v):
    g = generator(21)
    H, KVH = 16, 2
    cache = make(rt, 4, KVH, D)
    size = 2.0 ** torch.randint(-6, 7, (300, KVH, 1), generator=g, device=DEV)
    rt.kv_append([cache], [300], (randn(g, 300, KVH, D) * std_k).to(torch.bfloat16),
                 (randn(g, 300, KVH, D) * size * std_v).to(torch.bfloat16))
    q = (randn(g, 120, H, D) / std_k).to(torch.bfloat16)
    o = torch.empty_like(q)
    rt.gqa_attention_prefill(cache, q, None, H, 120, o)
    check(o, *attention(q, None, values(cache), 180))
    cache.close()


@pytest.mark.parametrize("rising", [True, False])
def test_tiles_of_very_different_size(rt, rising):
    """Values that grow or shrink by 2^63 over the tokens, most weight on any of them."""
    g = generator(22)
    H, KVH, D, n = 8, 1, 128, 320
    cache = make(rt, 4, KVH, D)
    step = torch.arange(n, device=DEV) // 32
    size = 2.0 ** (7.0 * (step if rising else step.flip(0)) - 35.0)
    k, v = bf16(g, n, KVH, D), (randn(g, n, KVH, D) * size[:, None, None]).to(torch.bfloat16)
    rt.kv_append([cache], [n], k, v)
    q = bf16(g, 100, H, D, std=3.0)
    o = torch.empty_like(q)
    rt.gqa_attention_prefill(cache, q, None, H, 100, o)
    check(o, *attention(q, None, values(cache), n - 100))
    cache.close()


# ---------------------------------------------------------------------------
# Long and wide calls
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,KVH,D,rd", [(16, 8, 128, 128), (8, 8, 64, 32), (12, 6, 256, 64)])
def test_long_appends_equal_short_ones(rt, H, KVH, D, rd, interleaved, bits):
    """Many pages in one call, whose workgroups take several KV heads, against pieces."""
    g = generator(30 + D)
    n = 6007
    one, many = make(rt, bits, KVH, D), make(rt, bits, KVH, D)
    for c in (one, many):
        fill(rt, c, generator(1), 11)
    q, k, v = (bf16(g, n, h, D) for h in (H, KVH, KVH))
    cfg = qm38.RotaryConfig(rd, interleaved, 1e4)
    out = torch.empty(2, n, H, D, dtype=torch.bfloat16, device=DEV)
    rt.kv_append([one], [n], k, v, rotary=cfg, q=q, q_out=out[0], num_heads=H)
    for a in range(0, n, 501):
        b = min(a + 501, n)
        rt.kv_append([many], [b - a], k[a:b], v[a:b], rotary=cfg, q=q[a:b], q_out=out[1, a:b], num_heads=H)
    assert torch.equal(out[0], out[1])
    equal(one, many)
    freq, factor = frequencies(rd, 1e4, "none", 1.0, 0, device=DEV)
    place = torch.arange(11, 11 + n, device=DEV)
    keys, vals = read(one)
    near_rows([a[11:] for a in keys], rotated(k, place, freq, factor, 0, interleaved))
    same_rows([a[11:] for a in vals], v.float())
    for c in (one, many):
        c.close()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", [1, 37, 64, 100, 128, 256])
def test_loads(rt, D, bits):
    """Ranges that begin and end anywhere, keys or values alone, outputs of any alignment."""
    g = generator(31 + D)
    KVH, n = 3, 75
    cache = make(rt, bits, KVH, D)
    fill(rt, cache, g, n)
    (k, _), (v, _) = values(cache)
    flat = torch.empty(2, n * KVH * D + 64, dtype=torch.bfloat16, device=DEV)
    for first, count in ((0, n), (0, 1), (n - 1, 1), (15, 2), (16, 16), (3, 60)):
        for shift in (0, 1, 8):
            flat.fill_(5.0)
            a, b = (x[shift:shift + count * KVH * D].view(count, KVH, D) for x in flat)
            cache.load(first, count, a, b if shift else None)
            if not shift:
                cache.load(first, count, None, b)
            for got, x in ((a, k), (b, v)):
                # (the cache's values are fp32 sums of one rounding, then bf16)
                assert torch.equal(got, x[first:first + count].float().to(torch.bfloat16))
            for x in flat:
                assert (x[:shift] == 5).all() and (x[shift + count * KVH * D:] == 5).all()
    cache.close()


@pytest.mark.parametrize("shape", [(16, 2, 64), (64, 8, 128), (26, 2, 128), (24, 4, 256), (32, 2, 256)])
def test_decode_of_64_sequences(rt, shape):
    g = generator(32)
    H, KVH, D = shape
    lengths = [(37 * b * b) % 1500 for b in range(64)]
    caches = [make(rt, 4, KVH, D) for _ in lengths]
    for c, n in zip(caches, lengths):
        if n:
            fill(rt, c, g, n)
    q, gate = bf16(g, 64, H, D, std=1.5), bf16(g, 64, H, D)
    k, v = randn(g, 64, KVH, D), randn(g, 64, KVH, D)
    o, again = torch.empty_like(q), torch.empty_like(q)
    rt.gqa_attention_q8(caches, q, gate, k, v, H, o)
    for b, c in enumerate(caches):
        assert c.sequence_length == lengths[b] + 1
        check(o[b:b + 1], *attention(q[b:b + 1], gate[b:b + 1], values(c), lengths[b]))
    rt.gqa_attention(caches, q, gate, H, o)
    rt.gqa_attention(caches, q, gate, H, again)
    assert torch.equal(o, again)
    for c in caches:
        c.close()


@pytest.mark.parametrize("shape,n", [((16, 1, 128), 20000), ((13, 1, 256), 9000), ((9, 1, 64), 40000), ((24, 4, 256), 70000)])
def test_decode_of_long_sequences(rt, shape, n):
    """Splits of many pages, up to 16 heads a KV head (two sets of columns)."""
    g = generator(33)
    H, KVH, D = shape
    cache = make(rt, 4, KVH, D)
    fill(rt, cache, g, n)
    q, k, v = bf16(g, 1, H, D, std=1.5), randn(g, 1, KVH, D), randn(g, 1, KVH, D)
    o = torch.empty_like(q)
    rt.gqa_attention_q8([cache], q, None, k, v, H, o)
    for part, x in zip(read(cache), (k, v)):
        same_rows([a[n:] for a in part], x)
    check(o, *attention(q, None, values(cache), n))
    cache.close()


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("H,KVH,D,rd", [(16, 4, 128, 128), (24, 4, 256, 64)])
def test_requests_served(rt, H, KVH, D, rd, bits):
    """Prompts of several requests in one append, their attention, then steps of the whole
    batch while one request ends, one is rolled back and one joins."""
    g = generator(40)
    cfg = qm38.RotaryConfig(rd, False, 1e6)
    freq, factor = frequencies(rd, 1e6, "none", 1.0, 0, device=DEV)
    caches = [make(rt, bits, KVH, D) for _ in range(4)]

    def append(which, counts):
        total = sum(counts)
        fused = bf16(g, total, (H + 2 * KVH) * D)
        q, k, v = fused.split([H * D, KVH * D, KVH * D], 1)
        out = torch.empty(total, H, D, dtype=torch.bfloat16, device=DEV)
        start = [c.sequence_length for c in which]
        rt.kv_append(which, counts, k, v, rotary=cfg, q=q, q_out=out, num_heads=H)
        place = torch.cat([torch.arange(s, s + n, device=DEV) for s, n in zip(start, counts)])
        turned = rotated(k.reshape(total, KVH, D), place, freq, factor, 0, False)
        first = 0
        for c, s, n in zip(which, start, counts):
            assert c.sequence_length == s + n
            if n:
                keys, vals = read(c)
                near_rows([a[s:] for a in keys], turned[first:first + n])
                same_rows([a[s:] for a in vals], v.reshape(total, KVH, D)[first:first + n].float())
            first += n
        return out

    counts = [300, 7, 0, 90]
    q = append(caches, counts)
    first = 0
    for c, n in zip(caches, counts):
        if n:
            mine = q[first:first + n]
            o = torch.empty_like(mine)
            rt.gqa_attention_prefill(c, mine, None, H, n, o)
            check(o, *attention(mine, None, values(c), 0))
        first += n
    live = [caches[0], caches[1], caches[3]]
    for step in range(20):
        if step == 5:
            live.append(caches[2])
        if step == 9:
            live[1].truncate(live[1].sequence_length - 4)
        if step == 13:
            live.pop(0)
        q = append(live, [1] * len(live))
        o = torch.empty_like(q)
        rt.gqa_attention(live, q, None, H, o)
        for b, c in enumerate(live):
            check(o[b:b + 1], *attention(q[b:b + 1], None, values(c), c.sequence_length - 1))
    for c in caches:
        c.close()


def test_decode_layers_over_a_4_bit_cache(rt, torch_dev):
    """A hybrid model's layers, as eager calls, as one call and as graph segments."""
    model = Model(rt, torch_dev, seed=11)

    def request():
        states, caches, descs = model.new_request()
        kept = []
        for i, d in enumerate(descs):
            if caches[i] is not None:
                caches[i] = rt.create_q4_kv_state(FULL["kv_heads"], FULL["head_dim"], 64)
                d.kv = caches[i].handle.value
                kept.append(caches[i])
        return states, caches, descs, kept

    h0 = _hidden0(1)
    _, _, descs, kv_a = request()
    states_b, caches_b, _, kv_b = request()
    _, _, descs_c, kv_c = request()
    st, st_c = _state_with(rt, torch_dev, h0), _state_with(rt, torch_dev, h0)
    hidden = torch.from_numpy(h0.copy()).to(torch_dev)
    graph = qm38.DecodeGraph(rt, st_c, descs_c, EPS)
    for t in range(5):
        rt.decode_layers(st, descs, _positions(t), EPS)
        _manual_token(rt, torch_dev, model, states_b, caches_b, hidden, _positions(t))
        graph.run(_positions(t))
        got = _hidden(rt, st)
        assert np.array_equal(got, hidden.cpu().numpy()), t
        assert np.array_equal(got, _hidden(rt, st_c)), t
    for a, b, c in zip(kv_a, kv_b, kv_c):
        assert a.sequence_length == 5 and a.bits == 4
        equal(a, b)
        equal(a, c)


def test_noalloc_equals_decode(rt):
    g = generator(41)
    H, KVH, D = 64, 8, 128
    for lengths in ([300, 5000, 17, 40000, 1], [260, 33], [5] * 40):
        a = [make(rt, 4, KVH, D) for _ in lengths]
        for c, n in zip(a, lengths):
            c.reserve(n + 1)
            fill(rt, c, g, n)
        b = [c.clone() for c in a]
        B = len(lengths)
        q, gate, k, v = bf16(g, B, H, D), bf16(g, B, H, D), randn(g, B, KVH, D), randn(g, B, KVH, D)
        want, got = torch.empty_like(q), torch.empty_like(q)
        rt.gqa_attention_q8(a, q, gate, k, v, H, want)
        rt.gqa_attention_q8_noalloc(b, q, gate, k, v, H, got)
        assert torch.equal(want, got)
        for x, y in zip(a, b):
            equal(x, y)
        for c in a + b:
            c.close()


def test_two_runtimes_on_their_streams(rt):
    """One runtime's cache appended to and read by another on another stream, in turn,
    with nothing between the calls."""
    g = generator(43)
    H, KVH, D = 16, 4, 128
    q, k, v = bf16(g, 400, H, D), bf16(g, 2400, KVH, D), bf16(g, 2400, KVH, D)
    plain = make(rt, 4, KVH, D)
    rt.kv_append([plain], [2400], k, v)
    want = torch.empty(2, 400, H, D, dtype=torch.bfloat16, device=DEV)
    rt.gqa_attention_prefill(plain, q, None, H, 400, want[0])
    rt.gqa_attention([plain], q[:1], None, H, want[1, :1])
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    r1, r2 = qm38.Runtime(0), qm38.Runtime(0)
    try:
        r1.set_stream(s1)
        r2.set_stream(s2)
        cache = r1.create_q4_kv_state(KVH, D)
        got, loaded = torch.empty_like(want), torch.empty(2400, KVH, D, dtype=torch.bfloat16, device=DEV)
        at = 0
        for i, n in enumerate((1000, 1, 399, 16, 984)):
            (r1, r2)[i % 2].kv_append([cache], [n], k[at:at + n], v[at:at + n])
            at += n
        r2.gqa_attention_prefill(cache, q, None, H, 400, got[0])
        r1.gqa_attention([cache], q[:1], None, H, got[1, :1])
        assert r2.lib.qm_kv_load(r2.handle, cache.handle, 0, 2400, loaded.data_ptr(), None) == 0
        cache.truncate(2000)
        r1.kv_append([cache], [400], k[2000:], v[2000:])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1, :1], want[1, :1])
        assert torch.equal(loaded, values(plain)[0][0].float().to(torch.bfloat16))
        equal(cache, plain)
        cache.close()
    finally:
        torch.cuda.synchronize()
        r1.close()
        r2.close()
        plain.close()


def test_partials_are_not_shared(rt):
    """Split attention of two runtimes on two streams at once: the partials are their own."""
    g = generator(44)
    H, KVH, D = 16, 4, 128
    streams, runtimes = [torch.cuda.Stream() for _ in range(2)], [qm38.Runtime(0) for _ in range(2)]
    jobs = []
    try:
        for s, r in zip(streams, runtimes):
            r.set_stream(s)
            cache = r.create_q4_kv_state(KVH, D)
            k, v = bf16(g, 9000, KVH, D), bf16(g, 9000, KVH, D)
            torch.cuda.synchronize()
            r.kv_append([cache], [9000], k, v)
            q = bf16(g, 50, H, D)
            torch.cuda.synchronize()
            want = torch.empty_like(q)
            r.gqa_attention_prefill(cache, q, None, H, 50, want)
            one = torch.empty_like(q[:1])
            r.gqa_attention([cache], q[:1], None, H, one)
            torch.cuda.synchronize()
            jobs.append((r, cache, q, want, one, torch.empty(6, *q.shape, dtype=q.dtype, device=DEV),
                         torch.empty(6, *one.shape, dtype=q.dtype, device=DEV)))
        for i in range(6):
            for r, cache, q, _, _, a, b in jobs:
                r.gqa_attention_prefill(cache, q, None, H, 50, a[i])
                r.gqa_attention([cache], q[:1], None, H, b[i])
        torch.cuda.synchronize()
        for _, cache, _, want, one, a, b in jobs:
            assert all(torch.equal(x, want) for x in a) and all(torch.equal(x, one) for x in b)
            cache.close()
    finally:
        torch.cuda.synchronize()
        for r in runtimes:
            r.close()


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def status(call, *args, **kw):
    with pytest.raises(qm38.QmError) as e:
        call(*args, **kw)
    return e.value.status


def test_refused_appends(rt):
    g = generator(50)
    H, KVH, D = 4, 2, 64
    a, b, other, wide = make(rt, 4, KVH, D), make(rt, 4, KVH, D), make(rt, 8, KVH, D), make(rt, 4, KVH, 128)
    full = make(rt, 4, KVH, D, max_tokens=20)
    k, v, q = bf16(g, 8, KVH, D), bf16(g, 8, KVH, D), bf16(g, 8, H, D)
    out = torch.full_like(q, 2.0)
    cfg = qm38.RotaryConfig(64, False, 1e4)
    pos = torch.zeros(9, dtype=torch.int32, device=DEV)
    shape, bad = "QM_ERR_INVALID_ATTENTION_SHAPE", "QM_ERR_INVALID_ARGUMENT"
    for c in (a, b, full):
        rt.kv_append([c], [8], k, v)
    was = [c.read() for c in (a, b, full)]
    for want, seqs, counts, kw in [
            (shape, [a, other], [4, 4], {}), (shape, [a, wide], [4, 4], {}), (bad, [a, b, a], [2, 2, 2], {}),
            ("QM_ERR_EMPTY_APPEND", [a, b], [0, 0], {}), ("QM_ERR_CAPACITY_EXCEEDED", [a, full], [1, 13], {}),
            ("QM_ERR_DIMENSION_OVERFLOW", [a], [(1 << 20) + 1], {}),
            (shape, [a], [8], dict(rotary=qm38.RotaryConfig(66, False, 1e4))),
            (shape, [a], [8], dict(rotary=qm38.RotaryConfig(60, False, 1e4), offset=6)),
            (shape, [a], [8], dict(rotary=qm38.RotaryConfig(7, False, 1e4))),
            (bad, [a], [8], dict(rotary=qm38.RotaryConfig(64, False, 0.5))),
            (bad, [a], [8], dict(q=q, q_out=out, num_heads=H)),
            ("QM_ERR_NULL_POINTER", [a], [8], dict(rotary=cfg, q=q, num_heads=H)),
            ("QM_ERR_EMPTY_DIMENSION", [a], [8], dict(rotary=cfg, q=q, q_out=out)),
            (bad, [a], [8], dict(rotary=cfg, q=q, q_out=k, num_heads=H)),
            (bad, [a], [8], dict(rotary=cfg, q=out.flatten()[:8 * 2 * D].view(8, 2, D),
                                 q_out=out.flatten()[64:64 + 8 * 2 * D].view(8, 2, D), num_heads=2)),
            ("QM_ERR_MISALIGNED", [a], [8], dict(rotary=cfg, positions=pos.data_ptr() + 2))]:
        assert status(rt.kv_append, seqs, counts, k, v, **kw) == want, (want, counts, kw)
    assert status(rt.kv_append, [a], [8], k.data_ptr() + 1, v) == "QM_ERR_MISALIGNED"
    narrow = torch.as_strided(k, (8, KVH, D), (64, D, 1))
    assert status(rt.kv_append, [a], [8], narrow, v) == bad
    # More workgroups than a launch takes (refused before anything grows or is read).
    for heads, dim in ((512, 1), (80, 256)):
        many = make(rt, 4, heads, dim)
        assert status(rt.kv_append, [many], [1 << 20], k.data_ptr(), v.data_ptr()) == "QM_ERR_DIMENSION_OVERFLOW"
        assert many.capacity_tokens < 1 << 20
        many.close()
    torch.cuda.synchronize()
    assert (out == 2).all()
    for c, old in zip((a, b, full), was):
        assert all(np.array_equal(x, y) for x, y in zip(c.read(), old))
    for c in (a, b, other, wide, full):
        c.close()


def test_refused_attention_and_loads(rt):
    g = generator(51)
    H, KVH, D = 4, 2, 64
    a, empty, other = make(rt, 4, KVH, D), make(rt, 4, KVH, D), make(rt, 8, KVH, D)
    fill(rt, a, g, 20)
    fill(rt, other, g, 20)
    q = bf16(g, 21, H, D)
    o = torch.full_like(q, 2.0)
    k = randn(g, 2, KVH, D)
    shape, bad, length = "QM_ERR_INVALID_ATTENTION_SHAPE", "QM_ERR_INVALID_ARGUMENT", "QM_ERR_INVALID_SEQUENCE_LENGTH"
    assert status(rt.gqa_attention, [a, empty], q, None, H, o) == length
    assert status(rt.gqa_attention, [a, other], q, None, H, o) == shape
    assert status(rt.gqa_attention_q8, [a, other], q, None, k, k, H, o) == shape
    assert status(rt.gqa_attention, [a, a], q, None, H, o) == bad
    assert status(rt.gqa_attention, [a], q, None, 3, o) == shape
    assert status(rt.gqa_attention, [a], q, None, 2 * 17, o) == shape
    assert status(rt.gqa_attention, [a], q.data_ptr() + 2, None, H, o) == "QM_ERR_MISALIGNED"
    assert status(rt.gqa_attention_prefill, a, q, None, H, 21, o) == length
    assert status(rt.gqa_attention_prefill, a, q, None, H, 0, o) == shape
    assert status(rt.gqa_attention_prefill, empty, q, None, H, 1, o) == length
    assert status(a.load, 0, 0, o, None) == "QM_ERR_EMPTY_DIMENSION"
    assert status(a.load, 1, 20, o, None) == length
    assert status(a.load, 0xFFFFFFFF, 2, o, None) == length
    assert status(a.load, 0, 2, None, None) == "QM_ERR_NULL_POINTER"
    assert status(a.load, 0, 2, o.data_ptr() + 1, None) == "QM_ERR_MISALIGNED"
    lib = rt.lib
    buf = np.zeros(20 * KVH * D, np.int8)
    assert lib.qm_kv_read(a.handle, buf.ctypes.data, None, None, None) != 0
    assert lib.qm_kv_read_q4(other.handle, buf.ctypes.data, None, None, None) != 0
    torch.cuda.synchronize()
    assert (o == 2).all() and a.sequence_length == 20 and empty.sequence_length == 0
    for c in (a, empty, other):
        c.close()


def test_calls_refused_under_capture(rt):
    """Calls that move a length or grow a buffer do not go into a graph, and the caches stay."""
    g = generator(52)
    H, KVH, D = 4, 2, 64
    cache = make(rt, 4, KVH, D)
    fill(rt, cache, g, 20)
    k, q = bf16(g, 1, KVH, D), bf16(g, 1, H, D)
    o = torch.empty_like(q)
    own, stream, graph = qm38.Runtime(0), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            own.set_stream(stream)
            o.fill_(4.0)
            assert status(own.kv_append, [cache], [1], k, k) == "QM_ERR_INVALID_ARGUMENT"
            assert status(own.gqa_attention, [cache], q, None, H, o) == "QM_ERR_INVALID_ARGUMENT"
            assert status(own.gqa_attention_prefill, cache, q, None, H, 1, o) == "QM_ERR_INVALID_ARGUMENT"
            assert own.lib.qm_kv_load(own.handle, cache.handle, 0, 1, o.data_ptr(), None) != 0
        graph.replay()
        torch.cuda.synchronize()
        assert (o == 4).all() and cache.sequence_length == 20
        assert own.lib.qm_runtime_set_stream(own.handle, C.c_void_p(2)) == 0  # the per-thread stream
        assert status(own.kv_append, [cache], [1], k, k) == "QM_ERR_INVALID_ARGUMENT"
    finally:
        own.set_stream(None)
        own.close()
        cache.close()
