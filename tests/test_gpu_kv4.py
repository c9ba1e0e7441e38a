"""GPU tests of the 4-bit KV cache, of appends that rotate on the way (both kinds of
cache), and of attention over them, against plain forms in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import qm38
from kv4_util import attention, check, frequencies, held, quantised, quantised8, read, rotated, spread, values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV) * std


def bf16(g, *shape, std=1.0):
    return randn(g, *shape, std=std).to(torch.bfloat16)


def make(rt, bits, KVH, D, **kw):
    return (rt.create_q4_kv_state if bits == 4 else rt.create_q8_kv_state)(KVH, D, **kw)


def fill(rt, cache, g, n):
    """n tokens whose keys have means of their own per channel."""
    KVH, D = cache.kv_heads, cache.head_dim
    k = (randn(g, n, KVH, D) + randn(g, KVH, D)).to(torch.bfloat16)
    v = bf16(g, n, KVH, D)
    rt.kv_append([cache], [n], k, v)
    return k, v


def same_rows(got, x):
    """A cache's content of one kind (read()) against quantised fp32 rows, bit for bit."""
    if len(got) == 2:
        codes, s = quantised8(x)
        assert torch.equal(got[0], codes)
        assert torch.equal(got[1], s)
        return
    codes, s, m = quantised(x)
    assert torch.equal(got[1].view(torch.int16), s.view(torch.int16))
    assert torch.equal(got[2].view(torch.int16), m.view(torch.int16))
    assert torch.equal(got[0], codes)


def near_rows(got, x):
    """The same of rotated rows x (float64), whose angles, position times frequency at
    up to 2^31, are known to 2^-21 (the frequency and the product round at 2^-53
    each): all that comes of rows within eps = 2^-20 of their largest element, which
    also covers the fp32 roundings on the way to a code (2^-23 of it at most)."""
    eps = x.abs().amax(-1, keepdim=True) * 2 ** -20
    if len(got) == 2:
        codes, s = got[0].double(), got[1].double()
        top = x.abs().amax(-1, keepdim=True)
        assert ((s - top / 127).abs() <= eps / 127 + 2 ** -126).all()
        low, high = (torch.round(((x + d) / s).clamp(-127, 127)) for d in (-eps, eps))
        assert ((codes >= low) & (codes <= high)).all()
        return
    codes, s, m = got
    groups = x.split(64, -1)
    for i, part in enumerate(groups):
        sg, mg, c = s[..., i:i + 1], m[..., i:i + 1], codes[..., 64 * i:64 * (i + 1)].double()
        low, high = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
        least, most = ((((high - low) + d) / 15).clamp(min=2 ** -126).to(torch.bfloat16) for d in (-2 * eps, 2 * eps))
        assert ((sg >= least) & (sg <= most)).all()
        least, most = ((low + 8 * sg.double() + d).to(torch.bfloat16) for d in (-eps, eps))
        assert ((mg >= least) & (mg <= most)).all()
        least, most = (torch.round(((part + d - mg.double()) / sg.double()).clamp(-8, 7)) for d in (-eps, eps))
        assert ((c >= least) & (c <= most)).all()


WIDTHS = [1, 37, 64, 65, 80, 128, 130, 200, 256]


# ---------------------------------------------------------------------------
# Appends
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", WIDTHS)
def test_append_quantises(rt, bits, D):
    """Codes, scales and offsets, and what they stand for read back."""
    g = generator(D)
    KVH, n = 3, 53
    cache = make(rt, bits, KVH, D)
    k, v = fill(rt, cache, g, n)
    for got, x in zip(read(cache), (k, v)):
        same_rows(got, x.float())
    out = [torch.full((n - 9, KVH, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    cache.load(5, n - 9, *out)
    for o, (x, _) in zip(out, values(cache)):
        assert torch.equal(o, x[5:n - 4].float().to(torch.bfloat16))
    only = torch.zeros_like(out[0])
    cache.load(5, n - 9, None, only)
    assert torch.equal(only, out[1])
    only.zero_()
    cache.load(5, n - 9, only, None)
    assert torch.equal(only, out[0])
    cache.close()


def test_error_of_codes(rt):
    """The bound that the header states."""
    g = generator(1)
    cache = make(rt, 4, 2, 256)
    for std, mean in ((1.0, 0.0), (1e-3, 5.0), (30.0, -1.0), (1e-20, 0.0)):
        cache.truncate(0)
        k = (randn(g, 200, 2, 256, std=std) + mean).to(torch.bfloat16)
        rt.kv_append([cache], [200], k, k)
        c, s, m = read(cache)[0]
        s, m = spread(s.double(), 256), spread(m.double(), 256)
        assert ((held(*read(cache)[0]) - k.double()).abs() <= s / 2 + s / 64 + m.abs() / 256).all()
    cache.close()


@pytest.mark.parametrize("D", [64, 80, 256])
def test_append_in_pieces(rt, D):
    """Rows in calls of any size, over pages that hold other tokens, after drops, and
    clones that go on by themselves: the content does not depend on it."""
    g = generator(2)
    KVH, n = 2, 77
    one, many = make(rt, 4, KVH, D), make(rt, 4, KVH, D)
    k, v = fill(rt, one, g, n)
    other = bf16(g, n, KVH, D)
    at = 0
    for step in (1, 1, 5, 9, 3, 14, 16, 1, 27):
        rt.kv_append([many], [min(step + 3, n)], other, other)  # dropped again
        many.truncate(at)
        rt.kv_append([many], [step], k[at:at + step], v[at:at + step])
        at += step
    assert at == n and many.sequence_length == n
    twin = many.clone()
    assert twin.bits == 4
    rt.kv_append([many], [7], other[:7], other[:7])
    for cache in (many, twin):
        cache.truncate(n)
        for a, b in zip(read(one), read(cache)):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    rt.kv_append([twin], [300], *(bf16(g, 300, KVH, D) for _ in range(2)))  # grows
    twin.truncate(n)
    for a, b in zip(read(one), read(twin)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for c in (one, many, twin):
        c.close()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D,rd,offset,interleaved,scaling", [
    (128, 128, 0, False, "none"), (128, 128, 0, True, "linear"), (256, 128, 0, False, "yarn"), (256, 64, 192, True, "none"),
    (64, 64, 0, False, "none"), (80, 80, 0, False, "linear"), (80, 80, 0, True, "none"), (37, 6, 3, False, "none"),
    (65, 10, 5, True, "yarn"), (130, 36, 4, False, "none"), (256, 256, 0, True, "none"), (256, 256, 0, False, "none"),
    (2, 2, 0, False, "none")])
def test_append_rotates(rt, bits, D, rd, offset, interleaved, scaling):
    """Keys and queries of a ragged batch from the rows of a fused projection."""
    g = generator(D + rd)
    KVH, H = 2, 6
    counts, cached = [5, 0, 33, 1, 16], [0, 3, 21, 16, 15]
    total = sum(counts)
    caches = [make(rt, bits, KVH, D) for _ in counts]
    for c, n in zip(caches, cached):
        if n:
            fill(rt, c, g, n)
    row = bf16(g, total, (H + 2 * KVH) * D + 24)
    q, k, v = row[:, :H * D], row[:, H * D:(H + KVH) * D], row[:, (H + KVH) * D:(H + 2 * KVH) * D]
    cfg = qm38.RotaryConfig(rd, interleaved, 1e4, scaling, 4.0, 64)
    freq, factor = frequencies(rd, 1e4, scaling, 4.0, 64, device=DEV)
    factor = torch.tensor(factor, dtype=torch.float32).item()
    at = torch.cat([torch.arange(n, device=DEV) + c for n, c in zip(counts, cached)])
    far = torch.randint(0, 2 ** 31 - 1, (total,), generator=g, device=DEV, dtype=torch.int32)
    before = [read(c) for c in caches]
    for positions in (None, far):
        for c, n in zip(caches, cached):
            c.truncate(n)
        place = at if positions is None else positions
        q_out = torch.full((total, H, D), 9.0, dtype=torch.bfloat16, device=DEV)
        rt.kv_append(caches, counts, k, v, rotary=cfg, positions=positions, q=q, q_out=q_out, num_heads=H, offset=offset)
        want = torch.empty_like(q_out)
        rt.rotary(cfg, [(q.contiguous(), want, H, D, offset)], total, positions=place.to(torch.int32))
        assert torch.equal(q_out, want)
        turned = rotated(k.reshape(total, KVH, D), place, freq, factor, offset, interleaved)
        first = 0
        for c, n, b, old in zip(caches, counts, cached, before):
            new = slice(first, first + n)
            first += n
            parts = read(c)
            for part, kept in zip(parts, old):
                assert all(torch.equal(a[:b], o) for a, o in zip(part, kept))
            if n:
                near_rows([a[b:] for a in parts[0]], turned[new])
                same_rows([a[b:] for a in parts[1]], v.reshape(total, KVH, D)[new].float())
    # In place, the rest of the rows untouched, and without keys' rotation.
    for c, n in zip(caches, cached):
        c.truncate(n)
    copy = row.clone()
    mine = copy[:, :H * D]
    rt.kv_append(caches, counts, k, v, rotary=cfg, positions=far, q=mine, q_out=mine, num_heads=H, offset=offset)
    assert torch.equal(mine.reshape(total, H, D), q_out)
    assert torch.equal(copy[:, H * D:], row[:, H * D:])
    for c, n in zip(caches, cached):
        c.truncate(n)
    rt.kv_append(caches, counts, k, v, positions=far)
    for part, x in zip(read(caches[2]), (k, v)):
        same_rows([a[21:] for a in part], x.reshape(total, KVH, D)[5:38].float())
    for c in caches:
        c.close()


def test_append_to_many_sequences(rt):
    """More sequences than one launch takes; 2-byte aligned rows."""
    g = generator(5)
    KVH, D, B = 2, 72, 64
    caches = [make(rt, 4, KVH, D) for _ in range(B)]
    counts = [(7 * b) % 5 for b in range(B)]
    total = sum(counts)
    flat = bf16(g, 2 * total * KVH * D + 1)[1:]
    k, v = flat.reshape(2, total, KVH, D)
    rt.kv_append(caches, counts, k, v)
    first = 0
    for c, n in zip(caches, counts):
        assert c.sequence_length == n
        if n:
            for part, x in zip(read(c), (k, v)):
                same_rows(part, x[first:first + n].float())
        first += n
        c.close()


@pytest.mark.parametrize("D", [64, 100, 256])
def test_special_values(rt, D):
    """Zeros, equal values, the largest and smallest, NaN and infinities: of their own group alone."""
    g = generator(6)
    KVH, n = 2, 20
    x = randn(g, n, KVH, D)
    x[0] = 0.0
    x[1] = 3.140625
    x[2] = 3.0e38
    x[3, 0, 0], x[3, 0, 1] = 3.0e38, -3.0e38
    x[4] *= 1e-40
    x[5, 1, 7] = math.nan
    x[6, 0, D - 1] = math.inf
    x[7, 1, 0] = -math.inf
    x[8, 0] = 1e-45
    x = x.to(torch.bfloat16)
    cache = make(rt, 4, KVH, D)
    rt.kv_append([cache], [n], x, x)
    for part in read(cache):
        same_rows(part, x.float())
    for part, _ in values(cache):
        assert (part[0] == 0).all() and (part[1] == 3.140625).all()
        nan = torch.isnan(part)
        want = torch.zeros_like(nan)
        want[5, 1, :64] = True
        want[6, 0, (D - 1) // 64 * 64:] = True
        want[7, 1, :64] = True
        assert torch.equal(nan, want)
    cache.close()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
SHAPES = [(8, 8, 64), (32, 8, 64), (16, 1, 64), (64, 8, 128), (20, 5, 80), (6, 2, 37), (12, 4, 100), (24, 4, 256), (7, 1, 200),
          (16, 1, 256), (3, 3, 1)]


def decode_case(rt, g, shape, lengths, gated=True, bits=4):
    """Caches of these lengths and a step's prepared rows."""
    H, KVH, D = shape
    caches = [make(rt, bits, KVH, D) for _ in lengths]
    for c, n in zip(caches, lengths):
        if n:
            fill(rt, c, g, n)
    B = len(lengths)
    q = bf16(g, B, H, D, std=1.5)
    gate = bf16(g, B, H, D) if gated else None
    k, v = randn(g, B, KVH, D), randn(g, B, KVH, D)
    return caches, q, gate, k, v


@pytest.mark.parametrize("lengths", [[0], [1], [15], [16], [500], [33, 0, 1, 4097, 700], [8000]])
@pytest.mark.parametrize("shape", SHAPES)
def test_decode(rt, shape, lengths):
    g = generator(sum(shape) + sum(lengths))
    H, KVH, D = shape
    caches, q, gate, k, v = decode_case(rt, g, shape, lengths, gated=sum(lengths) % 2 == 0)
    before = [read(c) for c in caches]
    o = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    rt.gqa_attention_q8(caches, q, gate, k, v, H, o)
    again = torch.empty_like(o)
    rt.gqa_attention(caches, q, gate, H, again)  # the tokens are there now
    for b, (c, n) in enumerate(zip(caches, lengths)):
        assert c.sequence_length == n + 1
        for part, old, x in zip(read(c), before[b], (k, v)):
            same_rows([a[n:] for a in part], x[b:b + 1])
            assert all(torch.equal(a[:n], o_) for a, o_ in zip(part, old))
        want, bound = attention(q[b:b + 1], None if gate is None else gate[b:b + 1], values(c), n)
        check(o[b:b + 1], want, bound)
        check(again[b:b + 1], want, bound)
    # A step after it, on the content as it is.
    rt.gqa_attention_q8(caches, q, gate, v, k, H, o)
    for b, (c, n) in enumerate(zip(caches, lengths)):
        want, bound = attention(q[b:b + 1], None if gate is None else gate[b:b + 1], values(c), n + 1)
        check(o[b:b + 1], want, bound)
        c.close()


@pytest.mark.parametrize("bits", [4, 8])
def test_decode_of_cached_tokens_in_a_large_batch(rt, bits):
    """More sequences than one launch takes, rows appended before; also the 8-bit cache."""
    g = generator(7)
    shape = H, KVH, D = (16, 4, 128)
    lengths = [1 + (37 * b) % 300 for b in range(40)] + [5000]
    caches, q, gate, _, _ = decode_case(rt, g, shape, lengths, bits=bits)
    o = torch.empty_like(q)
    rt.gqa_attention(caches, q, gate, H, o)
    for b, (c, n) in enumerate(zip(caches, lengths)):
        assert c.sequence_length == n
        want, bound = attention(q[b:b + 1], gate[b:b + 1], values(c), n - 1)
        check(o[b:b + 1], want, bound)
        c.close()


@pytest.mark.parametrize("rows,cached", [(1, 0), (2, 5), (5, 2001), (16, 16), (33, 15), (100, 0), (300, 1000)])
@pytest.mark.parametrize("shape", SHAPES)
def test_prefill(rt, shape, rows, cached):
    g = generator(sum(shape) + rows)
    H, KVH, D = shape
    cache = make(rt, 4, KVH, D)
    if cached:
        fill(rt, cache, g, cached)
    q, k, v = bf16(g, rows, H, D, std=1.5), randn(g, rows, KVH, D), randn(g, rows, KVH, D)
    gate = bf16(g, rows, H, D) if rows % 2 else None
    o = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    rt.gqa_attention_q8_prefill(cache, q, gate, k, v, H, rows, o)
    for part, x in zip(read(cache), (k, v)):
        same_rows([a[cached:] for a in part], x)
    want, bound = attention(q, gate, values(cache), cached)
    check(o, want, bound)
    o.fill_(7.0)
    rt.gqa_attention_prefill(cache, q, gate, H, rows, o)
    check(o, want, bound)
    assert cache.sequence_length == cached + rows
    cache.close()


def test_prefill_of_cached_tokens_8_bits(rt):
    g = generator(8)
    H, KVH, D = 12, 4, 100
    cache = make(rt, 8, KVH, D)
    fill(rt, cache, g, 777)
    q = bf16(g, 200, H, D, std=1.5)
    o = torch.empty_like(q)
    rt.gqa_attention_prefill(cache, q, None, H, 200, o)
    check(o, *attention(q, None, values(cache), 577))
    cache.close()


def test_dropped_tokens_leave_nothing(rt):
    """NaN and infinities in tokens that were dropped, in a page that is in use."""
    g = generator(9)
    shape = H, KVH, D = (8, 2, 128)
    caches, q, gate, k, v = decode_case(rt, g, shape, [37, 5])
    bad = torch.full((60, KVH, D), math.nan, dtype=torch.bfloat16, device=DEV)
    bad[::2] = math.inf
    rt.kv_append(caches, [30, 30], bad, bad)
    for c, n in zip(caches, (37, 5)):
        c.truncate(n)
    o = torch.empty_like(q)
    rt.gqa_attention(caches, q, gate, H, o)
    for b, (c, n) in enumerate(zip(caches, (37, 5))):
        check(o[b:b + 1], *attention(q[b:b + 1], gate[b:b + 1], values(c), n - 1))
    rt.gqa_attention_q8(caches, q, gate, k, v, H, o)
    for b, (c, n) in enumerate(zip(caches, (37, 5))):
        check(o[b:b + 1], *attention(q[b:b + 1], gate[b:b + 1], values(c), n))
    cache = caches[0]
    cache.truncate(37)
    qs = bf16(g, 9, H, D)
    os = torch.empty_like(qs)
    rt.gqa_attention_prefill(cache, qs, None, H, 9, os)
    check(os, *attention(qs, None, values(cache), 28))
    for c in caches:
        c.close()


def test_nan_reaches_who_sees_it(rt):
    """A NaN in a token's key or value: the rows that see it, their KV head, and (value) its group."""
    g = generator(10)
    H, KVH, D = 8, 2, 128
    for kind in (0, 1):
        cache = make(rt, 4, KVH, D)
        x = [bf16(g, 50, KVH, D) for _ in range(2)]
        x[kind][30, 1, 70] = math.nan
        rt.kv_append([cache], [50], *x)
        q = bf16(g, 40, H, D)
        o = torch.empty_like(q)
        rt.gqa_attention_prefill(cache, q, None, H, 40, o)  # row i is token 10 + i
        nan = torch.zeros(40, H, D, dtype=torch.bool, device=DEV)
        nan[20:, H // 2:, 64 * kind:] = True
        assert torch.equal(torch.isnan(o), nan)
        one = torch.empty_like(q[:1])
        rt.gqa_attention([cache], q[:1], None, H, one)
        assert torch.equal(torch.isnan(one), nan[-1:])
        cache.close()


@pytest.mark.parametrize("std_k,std_v", [(1e-12, 1e-12), (1.0, 1e20), (1e4, 1.0), (1.0, 1e-30), (1e-3, 1e36)])
def test_magnitudes(rt, std_k, std_v):
    """Keys, values and queries far from 1, and tokens of very different size side by side."""
    g = generator(11)
    H, KVH, D = 16, 2, 128
    cache = make(rt, 4, KVH, D)
    size = 2.0 ** torch.randint(-6, 7, (300, KVH, 1), generator=g, device=DEV)
    rt.kv_append([cache], [300], (randn(g, 300, KVH, D) * std_k).to(torch.bfloat16),
                 (randn(g, 300, KVH, D) * size * std_v).to(torch.bfloat16))
    q = (randn(g, 50, H, D) / std_k).to(torch.bfloat16)
    o = torch.empty_like(q)
    rt.gqa_attention_prefill(cache, q, None, H, 50, o)
    want, bound = attention(q, None, values(cache), 250)
    check(o, want, bound)
    one = torch.empty_like(q[:1])
    rt.gqa_attention([cache], q[-1:], None, H, one)
    check(one, want[-1:], bound[-1:])
    cache.close()


def test_a_cache_beyond_4_gb(rt):
    """Offsets that pass 32 bits, in the append, the reads and the attention."""
    g = generator(12)
    H, KVH, D = 16, 16, 256
    chunk, chunks = 65536, 16  # 4.8 GB
    cache = make(rt, 4, KVH, D)
    cache.reserve(chunk * chunks + 1)
    k, v = bf16(g, chunk, KVH, D), bf16(g, chunk, KVH, D)
    for i in range(chunks):
        rt.kv_append([cache], [chunk], k, v)
    tail = [bf16(g, 1, KVH, D) for _ in range(2)]
    rt.kv_append([cache], [1], *tail)
    out = [torch.empty(chunk, KVH, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    cache.load(chunk * (chunks - 1), chunk, *out)
    for got, x in zip(out, (k, v)):
        assert torch.equal(got, held(*quantised(x.float())).float().to(torch.bfloat16))
    q = bf16(g, 1, H, D)
    o = torch.empty_like(q)
    rt.gqa_attention([cache], q, None, H, o)
    heads = [0, 15]
    kv = []
    for x, t in zip((k, v), tail):
        x, t = (held(*quantised(y[:, heads].float())) for y in (x, t))
        kv.append(torch.cat([x] * chunks + [t]))
    want, bound = attention(q[:, heads], None, [(x, x.abs() + 1.0) for x in kv], chunk * chunks)
    check(o[:, heads], want, bound)
    cache.close()
