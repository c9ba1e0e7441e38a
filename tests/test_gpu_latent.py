"""GPU tests of rotary positions, the 8-bit latent cache and latent attention
against plain forms in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import qm38
from gpu_util import to_dev, tuned
from latent_util import HALF, assert_attention, attention, frequencies, quantised, rotated
from qm38 import synth

pytestmark = pytest.mark.gpu

EPS = 1e-6
WIDE, SMALL, ODD, TINY = (512, 64, 128, 128), (256, 32, 64, 64), (384, 48, 96, 80), (8, 8, 8, 8)


def bf16(gen, *shape, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda:0") * std).to(torch.bfloat16)


def generator(seed):
    g = torch.Generator(device="cuda:0")
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
def check_rotated(got, x, positions, freq, factor, offset, interleaved):
    ref = rotated(x, positions, freq, factor, offset, interleaved)
    rd = 2 * len(freq)
    inside = torch.zeros(x.shape[-1], dtype=torch.bool, device=x.device)
    inside[offset:offset + rd] = True
    assert torch.equal(got[..., ~inside], x[..., ~inside])
    # fp32 sine, cosine and products of the pair, then half a bf16 step.
    pair = rotated(x.abs(), torch.zeros_like(positions), freq, 1.0, offset, interleaved)
    size = (x.double().abs().amax() * factor) * 1e-6
    err = (got.double() - ref).abs()
    assert (err <= ref.abs() * HALF + size)[..., inside].all()
    assert pair.shape == ref.shape


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,width,offset,rd", [
    (1, 1, 2, 0, 2), (1, 20, 192, 128, 64), (5, 20, 192, 128, 64), (300, 3, 128, 0, 128), (7, 5, 65, 3, 30),
    (33, 2, 256, 0, 256), (2, 7, 96, 8, 24), (65, 64, 64, 16, 32)])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("yarn", 8.0)])
def test_rotary(rt, interleaved, rows, heads, width, offset, rd, scaling, factor):
    g = generator(rows + width)
    x = bf16(g, rows, heads, width)
    positions = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda:0", dtype=torch.int32)
    cfg = qm38.RotaryConfig(rd, interleaved, 1e6, scaling, factor, 4096)
    freq, mul = frequencies(rd, 1e6, scaling, factor, 4096, device="cuda:0")
    out = torch.full_like(x, 7.0)
    rt.rotary(cfg, [(x, out, heads, width, offset)], rows, positions=positions)
    check_rotated(out, x, positions, freq, mul, offset, interleaved)
    same = x.clone()
    rt.rotary(cfg, [(same, same, heads, width, offset)], rows, positions=positions)
    assert torch.equal(same, out)


def test_rotary_of_strided_tensors_in_one_launch(rt):
    """Queries and key inside one projection row, in place; the rest of the row stays."""
    g = generator(3)
    rows, H = 19, 6
    row = bf16(g, rows, H * 192 + 576 + 40)
    before = row.clone()
    base = 2 ** 32 - 19  # the last positions that fit
    cfg = qm38.RotaryConfig(64, True, 1e4)
    freq, _ = frequencies(64, 1e4, device="cuda:0")
    q, kv = row[:, :H * 192], row[:, H * 192:H * 192 + 576]
    s = row.shape[1]
    rt.rotary(cfg, [(q, q, H, 192, 128, s, s), (kv, kv, 1, 576, 512, s, s)], rows, position_base=base)
    positions = torch.arange(rows, device="cuda:0", dtype=torch.float64) + base
    check_rotated(q.reshape(rows, H, 192), before[:, :H * 192].reshape(rows, H, 192), positions, freq, 1.0, 128, True)
    check_rotated(kv[:, None], before[:, None, H * 192:H * 192 + 576], positions, freq, 1.0, 512, True)
    assert torch.equal(row[:, H * 192 + 576:], before[:, H * 192 + 576:])
    # From one column of a buffer to another: rows interleave, elements do not meet.
    out = torch.zeros(rows, 2, 64, dtype=torch.bfloat16, device="cuda:0")
    out[:, 0] = before[:, :64]
    rt.rotary(qm38.RotaryConfig(64), [(out[:, 0], out[:, 1], 1, 64, 0, 128, 128)], rows)
    positions = torch.arange(rows, device="cuda:0")
    check_rotated(out[:, 1:], before[:, None, :64], positions, freq, 1.0, 0, False)
    assert torch.equal(out[:, 0], before[:, :64])


def test_rotary_unaligned_equals_aligned(rt):
    g = generator(4)
    flat = bf16(g, 9 * 3 * 96 + 1)
    x = flat[1:].reshape(9, 3, 96)  # 2-byte aligned
    y, z = torch.empty_like(x), torch.empty_like(x)
    for interleaved in (False, True):
        cfg = qm38.RotaryConfig(32, interleaved)
        rt.rotary(cfg, [(x, y, 3, 96, 64)], 9, position_base=77)
        rt.rotary(cfg, [(x.clone(), z, 3, 96, 64)], 9, position_base=77)
        assert torch.equal(y, z)


def test_rotary_captured(rt):
    """A captured call replayed with other positions in its buffer, with eager calls between."""
    g = generator(5)
    x = bf16(g, 33, 8, 192)
    out = torch.empty_like(x)
    positions = torch.arange(33, device="cuda:0", dtype=torch.int32)
    cfg = qm38.RotaryConfig(64, True, 1e6, "yarn", 4.0, 8192)
    call = lambda o: rt.rotary(cfg, [(x, o, 8, 192, 128)], 33, positions=positions)  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    try:
        with torch.cuda.graph(graph, stream=stream):
            rt.set_stream(stream)
            call(out)
    finally:
        rt.set_stream(torch.cuda.current_stream())
    for i in range(4):
        positions += 1000 * i
        eager = torch.empty_like(x)
        call(eager)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


# ---------------------------------------------------------------------------
# The cache
# ---------------------------------------------------------------------------
def held(cache):
    """(latents, keys) float64 that a cache stands for."""
    codes, scales = (torch.from_numpy(a).to("cuda:0").double() for a in cache.read())
    return codes[:, :cache.rank] * scales[:, :1], codes[:, cache.rank:] * scales[:, 1:]


@pytest.mark.parametrize("widths", [WIDE, SMALL, ODD, TINY, (136, 64, 8, 8)])
@pytest.mark.parametrize("pieces", [(1,), (3, 1, 60, 1), (64,), (65, 400), (1000,)])
def test_cache_codes(rt, widths, pieces):
    rank, rope = widths[:2]
    g = generator(sum(pieces) + rank)
    cache = rt.create_latent_kv(rank, rope)
    rows = bf16(g, sum(pieces), rank + rope)
    rows[0] = 0  # the smallest scale
    rows[-1, rank:] *= 1e30
    at = 0
    for n in pieces:
        cache.append(rows[at:at + n].clone(), None, 0.0, n)
        at += n
    assert cache.sequence_length == at <= cache.capacity_tokens
    codes, scales = cache.read()
    for part, (lo, hi) in enumerate(((0, rank), (rank, rank + rope))):
        c, s = quantised(rows[:, lo:hi].double())
        assert np.array_equal(codes[:, lo:hi], c.cpu().numpy())
        assert np.array_equal(scales[:, part], s[:, 0].cpu().numpy())
    # Read back: the products rounded once.
    first = at // 3
    out = torch.empty(at - first, rank + rope, dtype=torch.bfloat16, device="cuda:0")
    cache.load(first, at - first, out)
    want = torch.cat([torch.from_numpy(codes[:, lo:hi]).float() * torch.from_numpy(scales[:, p:p + 1])
                      for p, (lo, hi) in enumerate(((0, rank), (rank, rank + rope)))], 1)[first:]
    assert torch.equal(out.cpu(), want.to(torch.bfloat16))


@pytest.mark.parametrize("n", [3, 5000])
def test_codes_between_two_steps(rt, n):
    """Quotients at a half and one bf16 step beside it, at scales of every size; rows
    with numbers that are none among them; 5000 rows end inside a wave's four."""
    g = generator(n)
    power = torch.randint(-100, 100, (n, 1), generator=g, device="cuda:0").double()
    half = torch.randint(0, 63, (n, 576), generator=g, device="cuda:0").double() + 0.5
    x = (half * torch.where(torch.rand((n, 576), generator=g, device="cuda:0") < 0.5, 1.0, -1.0)).to(torch.bfloat16)
    beside = (x.view(torch.int16) + torch.randint(-1, 2, (n, 576), generator=g, device="cuda:0").to(torch.int16)).view(torch.bfloat16)
    x = beside.double()
    x[:, 5], x[:, 520] = 127.0, -127.0  # the scale is the power of two
    rows = (x * 2.0 ** power).to(torch.bfloat16)
    rows[1, 3], rows[2, 570] = float("nan"), float("inf")
    cache = rt.create_latent_kv(512, 64)
    cache.append(rows, None, 0.0, n)
    codes, scales = cache.read()
    for part, (lo, hi) in enumerate(((0, 512), (512, 576))):
        c, s = quantised(rows[:, lo:hi].double())
        none = ~torch.isfinite(rows[:, lo:hi]).all(1).cpu().numpy()
        assert np.isnan(scales[none, part]).all() and (codes[none, lo:hi] == 0).all() and none.sum() == 1
        assert np.array_equal(codes[~none, lo:hi], c.cpu().numpy()[~none])
        assert np.array_equal(scales[~none, part], s[:, 0].cpu().numpy()[~none])


@pytest.mark.parametrize("widths", [WIDE, SMALL, ODD, TINY])
def test_cache_normalised(rt, widths):
    rank, rope = widths[:2]
    g = generator(rank)
    rows = bf16(g, 500, rank + rope, std=3.0)
    norm = torch.rand(rank, generator=g, device="cuda:0") + 0.5
    cache = rt.create_latent_kv(rank, rope)
    cache.append(rows, norm, EPS, 500)
    latent, key = held(cache)
    x = rows[:, :rank].double()
    x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * norm.double()
    # Half a step of the scale, and fp32's error of the norm (a few 2^-24 of the value).
    step = x.abs().amax(-1, keepdim=True) / 127
    assert ((latent - x).abs() <= step * (0.5 + 1e-4)).all()
    c, s = quantised(rows[:, rank:].double())
    assert torch.equal(key, c * s.double())


def test_cache_clone_truncate_reserve(rt):
    g = generator(9)
    rows = bf16(g, 300, 576)
    cache = rt.create_latent_kv(512, 64, max_tokens=300)
    cache.append(rows, None, 0.0, 100)
    copy = cache.clone()
    assert copy.sequence_length == 100 and copy.capacity_tokens == cache.capacity_tokens
    cache.truncate(10)
    cache.append(rows[200:], None, 0.0, 100)
    cache.reserve(190)
    assert cache.capacity_tokens == 300
    a, b = cache.read(), copy.read()
    assert np.array_equal(a[0][:10], b[0][:10]) and not np.array_equal(a[0][10:100], b[0][10:100])
    with pytest.raises(qm38.QmError) as e:
        cache.append(rows, None, 0.0, 191)
    assert e.value.status == "QM_ERR_CAPACITY_EXCEEDED" and cache.sequence_length == 110
    # The copy's bytes are its own.
    copy.append(rows[100:], None, 0.0, 200)
    whole = rt.create_latent_kv(512, 64)
    whole.append(rows, None, 0.0, 300)
    for x, y in zip(copy.read(), whole.read()):
        assert np.array_equal(x, y)
    for c in (cache, copy, whole):
        c.close()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def make_weights(rt, g, H, widths, std=None):
    rank, rope, nope, v = widths
    kv_b = bf16(g, H, nope + v, rank, std=rank ** -0.5 if std is None else std)
    scale = (nope + rope) ** -0.5
    return kv_b, scale, rt.create_latent_weights(qm38.LatentConfig(H, rank, nope, rope, v, scale), kv_b)


def filled(rt, g, widths, n, norm):
    rank, rope = widths[:2]
    cache = rt.create_latent_kv(rank, rope)
    if n:
        cache.append(bf16(g, n, rank + rope), norm, EPS, n)
    return cache


def check_decode(rt, widths, H, lengths, seed, q_std=1.5):
    rank, rope, nope, v = widths
    g = generator(seed)
    kv_b, scale, weights = make_weights(rt, g, H, widths)
    norm = torch.rand(rank, generator=g, device="cuda:0") + 0.5
    caches = [filled(rt, g, widths, n, norm) for n in lengths]
    B = len(lengths)
    q, kv = bf16(g, B, H, nope + rope, std=q_std), bf16(g, B, rank + rope)
    o = torch.full((B, H, v), float("nan"), dtype=torch.bfloat16, device="cuda:0")
    rt.latent_attention(weights, caches, q, kv, norm, EPS, o)
    for b, cache in enumerate(caches):
        assert cache.sequence_length == lengths[b] + 1
        latent, key = held(cache)
        ref, bound = attention(q[b:b + 1], latent, key, kv_b, nope, scale, lengths[b])
        assert_attention(o[b:b + 1], ref, bound, f"sequence {b} of {lengths[b]}")
    again = torch.empty_like(o)
    for cache, n in zip(caches, lengths):
        cache.truncate(n)
    rt.latent_attention(weights, caches, q, kv, norm, EPS, again)
    assert torch.equal(o, again)


@pytest.mark.parametrize("widths", [WIDE, SMALL, ODD, TINY, (128, 16, 24, 128), (264, 64, 128, 8)])
@pytest.mark.parametrize("H", [1, 5, 32, 33])
def test_decode_widths(rt, widths, H):
    check_decode(rt, widths, H, [0, 1, 31, 32, 63, 255, 256, 700], H)


@pytest.mark.parametrize("H,lengths", [(128, [4097]), (64, [20000, 3, 8191]), (20, [70001]), (8, [5] * 64),
                                       (16, [2047, 2048, 2049])])
def test_decode_lengths(rt, H, lengths):
    check_decode(rt, WIDE, H, lengths, H)


@pytest.mark.parametrize("widths,H,lengths", [(TINY, 1024, [100, 0, 33]), (SMALL, 1024, [70]), (TINY, 1024, list(range(64))),
                                              (WIDE, 1023, [2000])])
def test_decode_most_heads(rt, widths, H, lengths):
    check_decode(rt, widths, H, lengths, H + len(lengths))


def test_decode_peaked(rt):
    """Scores of some hundreds: one token takes almost all of a row, the running
    maximum rises through the cache and falls behind."""
    check_decode(rt, SMALL, 40, [3000, 10], 1, q_std=60.0)


def check_prefill(rt, widths, H, cached, rows, seed, q_std=1.5):
    rank, rope, nope, v = widths
    g = generator(seed)
    kv_b, scale, weights = make_weights(rt, g, H, widths)
    norm = torch.rand(rank, generator=g, device="cuda:0") + 0.5
    cache = filled(rt, g, widths, cached, norm)
    q, kv = bf16(g, rows, H, nope + rope, std=q_std), bf16(g, rows, rank + rope)
    o = torch.full((rows, H, v), float("nan"), dtype=torch.bfloat16, device="cuda:0")
    rt.latent_attention_prefill(weights, cache, q, kv, norm, EPS, rows, o)
    assert cache.sequence_length == cached + rows
    latent, key = held(cache)
    ref, bound = attention(q, latent, key, kv_b, nope, scale, cached)
    assert_attention(o, ref, bound, f"{rows} rows on {cached}")
    cache.truncate(cached)
    again = torch.empty_like(o)
    rt.latent_attention_prefill(weights, cache, q, kv, norm, EPS, rows, again)
    assert torch.equal(o, again)


FORMS = {"absorbed": dict(QM38_LATENT_FORM=1), "expanded": dict(QM38_LATENT_FORM=2),
         "head by head": dict(QM38_LATENT_FORM=2, QM38_LATENT_MB=1)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("widths", [WIDE, SMALL, ODD, TINY, (200, 8, 128, 40), (512, 64, 64, 128)])
@pytest.mark.parametrize("H,cached,rows", [(1, 0, 1), (5, 0, 33), (3, 1000, 7), (20, 31, 130), (33, 64, 65)])
def test_prefill_widths(torch_dev, form, widths, H, cached, rows):
    with tuned(**FORMS[form]) as rt:
        check_prefill(rt, widths, H, cached, rows, H + rows)


@pytest.mark.parametrize("H,cached,rows", [(32, 20001, 5), (64, 0, 300), (8, 4096, 513), (128, 100, 40), (2, 0, 2000)])
def test_prefill_sizes(rt, H, cached, rows):
    check_prefill(rt, WIDE, H, cached, rows, H + rows)


# Workgroups of eight waves, of one end (300 rows of 130 heads) or both ends of the
# prompt (520 of 66, whose middle has one, 250 of 130), and of four; rows end inside a
# wave, a workgroup and a tile.
@pytest.mark.parametrize("widths", [WIDE, SMALL, (128, 64, 64, 128), (128, 64, 128, 64)])
@pytest.mark.parametrize("H,cached,rows", [(130, 20, 300), (66, 1, 520), (130, 7, 250), (20, 333, 300), (1, 0, 1025)])
def test_prefill_workgroups(torch_dev, widths, H, cached, rows):
    with tuned(QM38_LATENT_FORM=2) as rt:
        check_prefill(rt, widths, H, cached, rows, H + rows)


# Columns' groups that fill the chip once with one split (160), more than once
# (1280), and with 9 splits and more.
@pytest.mark.parametrize("H,cached,rows", [(20, 3000, 512), (20, 100, 4096), (64, 2500, 24), (2, 0, 700)])
def test_absorbed_splits(torch_dev, H, cached, rows):
    with tuned(QM38_LATENT_FORM=1) as rt:
        check_prefill(rt, SMALL, H, cached, rows, H + rows)


def test_cache_beyond_32_bit_offsets(rt):
    """7.5 million tokens, 4.4 GB of codes: all but the last hundred alike, so that
    the softmax over them is that over 101 tokens, one of them weighing 7.5 million."""
    rank, rope, nope, v = WIDE
    g = generator(31)
    H, alike, chunk = 8, 7_500_000, 500_000
    kv_b, scale, weights = make_weights(rt, g, H, WIDE)
    one, others = bf16(g, 1, rank + rope, std=0.01), bf16(g, 100, rank + rope)
    cache, few = rt.create_latent_kv(rank, rope), rt.create_latent_kv(rank, rope)
    cache.reserve(alike + 100)
    many = one.expand(chunk, -1).contiguous()
    for _ in range(alike // chunk):
        cache.append(many, None, 0.0, chunk)
    cache.append(others, None, 0.0, 97)
    few.append(torch.cat([one, others]), None, 0.0, 101)
    latent, key = held(few)
    w = kv_b.double()
    k, values = latent @ w[:, :nope].transpose(1, 2), latent @ w[:, nope:].transpose(1, 2)  # [H][101][nope], [H][101][v]
    weigh = torch.zeros(101, dtype=torch.float64, device="cuda:0")
    weigh[0] = np.log(alike)
    q = bf16(g, 3, H, nope + rope, std=8.0)
    x = q.double().transpose(0, 1)
    score = (x[..., :nope] @ k.transpose(1, 2) + x[..., nope:] @ key.T) * scale + weigh  # [H][3][101]
    o = torch.empty(3, H, v, dtype=torch.bfloat16, device="cuda:0")
    rt.latent_attention(weights, [cache], q[:1], others[97:98], None, 0.0, o[:1])
    rt.latent_attention_prefill(weights, cache, q[1:], others[98:], None, 0.0, 2, o[1:])
    assert cache.sequence_length == alike + 100
    for row in range(3):
        p = torch.softmax(score[:, row:row + 1, :99 + row], -1)
        assert 0.01 < float(p[..., 1:].sum(-1).mean()) < 0.99  # both kinds count
        ref = (p @ values[:, :99 + row]).transpose(0, 1)
        assert_attention(o[row:row + 1], ref, torch.full_like(ref, torch.inf), f"row {row}")
    out = torch.empty(1, rank + rope, dtype=torch.bfloat16, device="cuda:0")
    near = torch.empty_like(out)
    cache.load(alike + 50, 1, out)
    few.load(51, 1, near)
    assert torch.equal(out, near)
    cache.close()

@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("widths,H,cached,rows", [(TINY, 1024, 5, 70), (SMALL, 1000, 0, 40)])
def test_prefill_most_heads(torch_dev, form, widths, H, cached, rows):
    with tuned(**FORMS[form]) as rt:
        check_prefill(rt, widths, H, cached, rows, H + rows)


@pytest.mark.parametrize("form", FORMS)
def test_prefill_peaked(torch_dev, form):
    with tuned(**FORMS[form]) as rt:
        check_prefill(rt, ODD, 12, 700, 300, 2, q_std=60.0)


@pytest.mark.parametrize("form", FORMS)
def test_scales_far_apart(torch_dev, form):
    """Tokens whose latents and keys are 2^-40 to 2^40 times others', and tokens
    of zeros, alone in a tile and beside others."""
    rank, rope, nope, v = SMALL
    with tuned(**FORMS[form]) as rt:
        g = generator(18)
        H, rows = 6, 200
        kv_b, scale, weights = make_weights(rt, g, H, SMALL)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        kv[:40] = 0
        kv[50:60, :rank] = 0
        kv[60:70, rank:] = 0
        kv[70:75] *= 2.0 ** -40
        kv[100, :rank] *= 2.0 ** 40
        q[110:115] *= 2.0 ** -30
        q[116] *= 2.0 ** 20
        kv[150:152, :rank] *= 2.0 ** 20
        cache = rt.create_latent_kv(rank, rope)
        o = torch.full((rows, H, v), float("nan"), dtype=torch.bfloat16, device=torch_dev)
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
        latent, key = held(cache)
        ref, bound = attention(q, latent, key, kv_b, nope, scale, 0)
        err = (o.double() - ref).abs()
        assert (err <= bound + 1e-30).all(), float((err / (bound + 1e-30)).max())
        assert (o[:40] == 0).all()


@pytest.mark.parametrize("form", FORMS)
def test_a_large_token_that_is_not_attended(torch_dev, form):
    """A token whose latent is 2^20 times the others' but whose score leaves it
    nothing (the shared key's part decides) costs the others no precision, and
    rows that do not see it none either."""
    rank, rope, nope, v = SMALL
    with tuned(**FORMS[form]) as rt:
        g = generator(19)
        H, rows = 6, 200
        kv_b, scale, weights = make_weights(rt, g, H, SMALL)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        q[..., :nope] = 0
        q[..., nope:] = 1
        kv[5, :rank] *= 2.0 ** 20
        kv[110, :rank] *= 2.0 ** 20
        kv[[5, 110], rank:] = -100.0
        cache = rt.create_latent_kv(rank, rope)
        o = torch.full((rows, H, v), float("nan"), dtype=torch.bfloat16, device=torch_dev)
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
        latent, key = held(cache)
        ref, bound = attention(q, latent, key, kv_b, nope, scale, 0)
        assert_attention(o, ref, bound)


def test_prefill_in_pieces_equals_decode_steps(rt):
    """A prompt in two chunks and tokens decoded one by one leave the same cache;
    their outputs agree with one prefill of all rows within both forms' bounds."""
    rank, rope, nope, v = WIDE
    g = generator(11)
    H, rows = 20, 230
    kv_b, scale, weights = make_weights(rt, g, H, WIDE)
    norm = torch.rand(rank, generator=g, device="cuda:0") + 0.5
    q, kv = bf16(g, rows, H, nope + rope, std=1.5), bf16(g, rows, rank + rope)
    o = torch.empty(rows, H, v, dtype=torch.bfloat16, device="cuda:0")
    whole, parts = rt.create_latent_kv(rank, rope), rt.create_latent_kv(rank, rope)
    rt.latent_attention_prefill(weights, whole, q, kv, norm, EPS, rows, o)
    p = torch.empty_like(o)
    for lo, hi in ((0, 200), (200, 220)):
        rt.latent_attention_prefill(weights, parts, q[lo:hi].clone(), kv[lo:hi].clone(), norm, EPS, hi - lo, p[lo:hi])
    for i in range(220, rows):
        rt.latent_attention(weights, [parts], q[i:i + 1].clone(), kv[i:i + 1].clone(), norm, EPS, p[i:i + 1])
    for x, y in zip(whole.read(), parts.read()):
        assert np.array_equal(x, y)
    latent, key = held(whole)
    ref, bound = attention(q, latent, key, kv_b, nope, scale, 0)
    assert_attention(o, ref, bound, "whole")
    assert_attention(p, ref, bound, "pieces")


def test_weights_from_q4(rt, torch_dev):
    """kv_b as a Q4 job gives what its values rounded to bf16 give."""
    rank, rope, nope, v = 256, 64, 64, 48
    H = 6
    rng = np.random.default_rng(12)
    g = generator(12)
    mat = synth.q4_matrix(rng, H * (nope + v), rank)
    job = qm38.Runtime.job(*(to_dev(a, torch_dev) for a in mat), mat[0].shape[0])
    w = synth.unpack_q4(mat[0]).astype(np.float32).reshape(-1, rank // 64, 64)
    w = w * synth.bf16_to_f32(mat[1])[..., None] + synth.bf16_to_f32(mat[2])[..., None]
    plain = torch.from_numpy(w.reshape(H, nope + v, rank)).to(torch.bfloat16).to(torch_dev)
    cfg = qm38.LatentConfig(H, rank, nope, rope, v, 0.1)
    outs = []
    q, kv = bf16(g, 40, H, nope + rope), bf16(g, 40, rank + rope)
    for source in (job, plain):
        weights = rt.create_latent_weights(cfg, source)
        cache = rt.create_latent_kv(rank, rope)
        o = torch.empty(40, H, v, dtype=torch.bfloat16, device=torch_dev)
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, 40, o)
        outs.append(o)
    assert torch.equal(*outs)


@pytest.mark.parametrize("form", FORMS)
def test_numbers_that_are_none(torch_dev, form):
    with tuned(**FORMS[form]) as rt:
        check_numbers_that_are_none(rt)


def check_numbers_that_are_none(rt):
    """A token whose row holds an infinity or NaN poisons the rows that see it,
    and no other; a query that does poisons its own row and head."""
    rank, rope, nope, v = SMALL
    g = generator(13)
    H, rows = 5, 40
    kv_b, scale, weights = make_weights(rt, g, H, SMALL)
    q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
    kv[30, 3] = float("inf")
    kv[35, rank + 2] = float("-inf")
    q[7, 2, 5] = float("nan")
    q[9, 1, nope + 3] = float("inf")
    cache = rt.create_latent_kv(rank, rope)
    o = torch.zeros(rows, H, v, dtype=torch.bfloat16, device="cuda:0")
    rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
    bad = torch.isnan(o).all(-1)
    want = torch.zeros_like(bad)
    want[30:] = True
    want[7, 2] = want[9, 1] = True
    assert torch.equal(bad, want)
    assert torch.equal(torch.isfinite(o).all(-1), ~want)


def test_streams_in_turn(torch_dev):
    """Calls of one runtime on several streams share its workspaces; each gives
    what it gives alone."""
    rank, rope, nope, v = SMALL
    with tuned() as rt:
        g = generator(14)
        H = 8
        kv_b, scale, weights = make_weights(rt, g, H, SMALL)
        streams = [torch.cuda.Stream() for _ in range(3)]
        caches = [filled(rt, g, SMALL, 900 + 100 * i, None) for i in range(3)]
        q, kv = bf16(g, 3, H, nope + rope), bf16(g, 3, rank + rope)
        alone, outs = [], [[torch.empty(1, H, v, dtype=torch.bfloat16, device=torch_dev) for _ in range(6)] for _ in range(3)]
        for i, cache in enumerate(caches):
            o = torch.empty(1, H, v, dtype=torch.bfloat16, device=torch_dev)
            rt.latent_attention(weights, [cache], q[i:i + 1].clone(), kv[i:i + 1].clone(), None, 0.0, o)
            cache.truncate(cache.sequence_length - 1)
            alone.append(o)
        qs, kvs = [q[i:i + 1].clone() for i in range(3)], [kv[i:i + 1].clone() for i in range(3)]
        busy = torch.randn(2048, 2048, device=torch_dev)
        torch.cuda.synchronize()
        for s in streams:
            with torch.cuda.stream(s):
                busy @ busy
        for r in range(6):
            for i, s in enumerate(streams):
                rt.set_stream(s)
                rt.latent_attention(weights, [caches[i]], qs[i], kvs[i], None, 0.0, outs[i][r])
                caches[i].truncate(caches[i].sequence_length - 1)
        torch.cuda.synchronize()
        rt.set_stream(torch.cuda.current_stream())
        for i in range(3):
            for o in outs[i]:
                assert torch.equal(o, alone[i])


def test_cache_used_from_another_runtime(rt, torch_dev):
    """The owner's append comes before another runtime's attention, and after it the owner's read."""
    rank, rope, nope, v = SMALL
    with tuned() as other:
        other.set_stream(torch.cuda.Stream())
        g = generator(15)
        kv_b, scale, weights = make_weights(rt, g, 4, SMALL)
        q, kv = bf16(g, 1, 4, nope + rope), bf16(g, 1, rank + rope)
        rows = bf16(g, 5000, rank + rope)
        o = torch.empty(1, 4, v, dtype=torch.bfloat16, device=torch_dev)
        torch.cuda.synchronize()
        cache = rt.create_latent_kv(rank, rope)
        cache.append(rows, None, 0.0, 5000)
        other.latent_attention(weights, [cache], q, kv, None, 0.0, o)
        latent, key = held(cache)
        torch.cuda.synchronize()
        ref, bound = attention(q, latent, key, kv_b, nope, scale, 5000)
        assert_attention(o, ref, bound)


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def refused(status, call, *args, **kw):
    with pytest.raises(qm38.QmError) as e:
        call(*args, **kw)
    assert e.value.status == status, e.value


def test_refusals(rt):
    rank, rope, nope, v = SMALL
    g = generator(16)
    kv_b, scale, weights = make_weights(rt, g, 4, SMALL)
    q, kv = bf16(g, 2, 4, nope + rope), bf16(g, 2, rank + rope)
    o = torch.empty(2, 4, v, dtype=torch.bfloat16, device="cuda:0")
    a, b, wide = rt.create_latent_kv(rank, rope), rt.create_latent_kv(rank, rope), rt.create_latent_kv(512, rope)
    refused("QM_ERR_INVALID_ARGUMENT", rt.latent_attention, weights, [a, a], q, kv, None, 0.0, o)
    refused("QM_ERR_INVALID_ARGUMENT", rt.latent_attention, weights, [], q, kv, None, 0.0, o)
    refused("QM_ERR_INVALID_ATTENTION_SHAPE", rt.latent_attention, weights, [a, wide], q, kv, None, 0.0, o)
    refused("QM_ERR_NULL_POINTER", rt.latent_attention, weights, [a, b], q, None, None, 0.0, o)
    refused("QM_ERR_MISALIGNED", rt.latent_attention, weights, [a, b], q.data_ptr() + 2, kv, None, 0.0, o)
    refused("QM_ERR_INVALID_ARGUMENT", rt.latent_attention, weights, [a, b], q, kv, kv_b.float(), -1.0, o)
    refused("QM_ERR_INVALID_ATTENTION_SHAPE", rt.latent_attention_prefill, weights, a, q, kv, None, 0.0, 0, o)
    refused("QM_ERR_EMPTY_APPEND", a.append, kv, None, 0.0, 0)
    refused("QM_ERR_INVALID_SEQUENCE_LENGTH", a.load, 0, 1, kv)
    refused("QM_ERR_INVALID_SEQUENCE_LENGTH", a.truncate, 1)
    refused("QM_ERR_DIMENSION_OVERFLOW", a.reserve, 2 ** 32 - 1)
    for bad in ((0, rank, nope, rope, v), (4, 520, nope, rope, v), (4, rank, 136, rope, v), (4, rank, nope, 72, v),
                (4, rank, nope, rope, 12)):
        refused("QM_ERR_INVALID_ATTENTION_SHAPE", rt.create_latent_weights, qm38.LatentConfig(*bad, 1.0), kv_b)
    refused("QM_ERR_INVALID_ARGUMENT", rt.create_latent_weights,
            qm38.LatentConfig(4, rank, nope, rope, v, float("nan")), kv_b)
    job = qm38.Runtime.job(kv_b, kv_b, kv_b, 100)
    refused("QM_ERR_WRONG_LENGTH", rt.create_latent_weights, qm38.LatentConfig(4, rank, nope, rope, v, 1.0), job)
    refused("QM_ERR_INPUT_NOT_GROUPED", rt.create_latent_weights, qm38.LatentConfig(4, 264, nope, rope, v, 1.0), job)
    # A failed call leaves the lengths.
    small = rt.create_latent_kv(rank, rope, max_tokens=1)
    small.append(kv, None, 0.0, 1)
    refused("QM_ERR_CAPACITY_EXCEEDED", rt.latent_attention, weights, [a, small], q, kv, None, 0.0, o)
    assert (a.sequence_length, small.sequence_length) == (0, 1)


def test_capture_is_refused(torch_dev):
    """The calls that move a cache's length do not go into a graph, and say so."""
    rank, rope, nope, v = SMALL
    with tuned() as rt:
        g = generator(17)
        kv_b, scale, weights = make_weights(rt, g, 4, SMALL)
        q, kv = bf16(g, 1, 4, nope + rope), bf16(g, 1, rank + rope)
        o = torch.empty(1, 4, v, dtype=torch.bfloat16, device=torch_dev)
        cache = filled(rt, g, SMALL, 10, None)
        x = torch.zeros(4, device=torch_dev)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            rt.set_stream(stream)
            x += 1
            refused("QM_ERR_INVALID_ARGUMENT", rt.latent_attention, weights, [cache], q, kv, None, 0.0, o)
            refused("QM_ERR_INVALID_ARGUMENT", rt.latent_attention_prefill, weights, cache, q, kv, None, 0.0, 1, o)
            refused("QM_ERR_INVALID_ARGUMENT", cache.append, kv, None, 0.0, 1)
            refused("QM_ERR_INVALID_ARGUMENT", cache.load, 0, 1, kv)
        rt.set_stream(torch.cuda.current_stream())
        graph.replay()
        rt.latent_attention(weights, [cache], q, kv, None, 0.0, o)
        torch.cuda.synchronize()
        assert cache.sequence_length == 11 and float(x[0]) == 1.0


def test_more_rows_than_a_launch_takes(rt):
    """2^23 + 5 rows turned, 2^22 + 5 appended and read back: the rows at the ends
    and where one launch follows another."""
    n = (1 << 23) + 5
    g = generator(41)
    x = bf16(g, n, 1, 8)
    y = torch.empty_like(x)
    rt.rotary(qm38.RotaryConfig(4, interleaved=True, theta=100.0), [(x, y, 1, 8, 2)], n, position_base=7)
    freq, factor = frequencies(4, 100.0, device="cuda:0")
    for lo in (0, (1 << 23) - 4, n - 4):
        check_rotated(y[lo:lo + 4], x[lo:lo + 4], torch.arange(lo + 7, lo + 11, device="cuda:0"), freq, factor, 2, True)
    n = (1 << 22) + 5
    rows = x[:n, 0].repeat(1, 2).contiguous()  # rank 8, rope_dim 8
    cache = rt.create_latent_kv(8, 8)
    cache.append(rows, None, 0.0, n)
    assert cache.sequence_length == n
    out = torch.empty_like(rows)
    cache.load(0, n, out)
    c, s = quantised(rows[:, :8].double())
    want = (c * s.double()).to(torch.bfloat16)
    assert torch.equal(out[:, :8], want) and torch.equal(out[:, 8:], want)
    cache.close()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("widths", [WIDE, ODD])
def test_output_of_any_alignment(torch_dev, form, widths):
    """An o on 2 bytes holds what an aligned one does, and nothing around it changes."""
    rank, rope, nope, v = widths
    H, rows = 6, 70
    with tuned(**FORMS[form]) as rt:
        g = generator(43)
        _, _, weights = make_weights(rt, g, H, widths)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        outs = []
        for shift in (0, 1):
            flat = torch.full((rows * H * v + 16,), 7.0, dtype=torch.bfloat16, device=torch_dev)
            o = flat[8 + shift:8 + shift + rows * H * v].view(rows, H, v)
            cache = rt.create_latent_kv(rank, rope)
            rt.latent_attention_prefill(weights, cache, q[:rows - 1], kv[:rows - 1], None, 0.0, rows - 1, o[:rows - 1])
            rt.latent_attention(weights, [cache], q[rows - 1:].clone(), kv[rows - 1:].clone(), None, 0.0, o[rows - 1:])
            rt.synchronize()
            outs.append(o.clone())
            assert (flat[:8 + shift] == 7).all() and (flat[8 + shift + rows * H * v:] == 7).all()
            cache.close()
        assert torch.equal(*outs)


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [19, 300])
def test_a_layer_of_them(rt, torch_dev, rows):
    """Quantised projections, positions turned in place, the latent cache and its
    attention, the output projection: a prompt, then two sequences decoded together.
    Each operator against its formula on what the one before it gave."""
    E, H = 512, 12
    rank, rope, nope, v = 256, 64, 64, 64
    rng, g = np.random.default_rng(21), generator(21)

    def matrix(n, k):
        mat = synth.q4_matrix(rng, n, k)
        w = synth.unpack_q4(mat[0]).astype(np.float32).reshape(-1, k // 64, 64)
        w = w * synth.bf16_to_f32(mat[1])[..., None] + synth.bf16_to_f32(mat[2])[..., None]
        dev = tuple(to_dev(a, torch_dev) for a in mat)
        return dev, qm38.Runtime.job(*dev, n), torch.from_numpy(w.reshape(n, k)).to(torch_dev).double()

    held_q, q_job, _ = matrix(H * (nope + rope), E)
    held_kv, kv_job, _ = matrix(rank + rope, E)
    held_b, b_job, b_plain = matrix(H * (nope + v), rank)
    held_o, o_job, o_plain = matrix(E, H * v)
    norm = torch.rand(rank, generator=g, device=torch_dev) + 0.5
    scale = (nope + rope) ** -0.5
    weights = rt.create_latent_weights(qm38.LatentConfig(H, rank, nope, rope, v, scale), b_job)
    kv_b = b_plain.to(torch.bfloat16).reshape(H, nope + v, rank)
    turn = qm38.RotaryConfig(rope, interleaved=True, theta=1e4)
    freq, factor = frequencies(rope, 1e4, device=torch_dev)

    def layer(x, positions, attend):
        n = x.shape[0]
        q = torch.empty(n, H, nope + rope, dtype=torch.bfloat16, device=torch_dev)
        kv = torch.empty(n, rank + rope, dtype=torch.bfloat16, device=torch_dev)
        rt.q4_project([q_job, kv_job], x, E, n, [q, kv])
        rt.synchronize()
        before = q.clone(), kv.clone()
        rt.rotary(turn, [(q, q, H, nope + rope, nope), (kv, kv, 1, rank + rope, rank)], n, positions=positions)
        o = torch.empty(n, H, v, dtype=torch.bfloat16, device=torch_dev)
        attend(q, kv, o)
        y = torch.empty(n, E, dtype=torch.bfloat16, device=torch_dev)
        rt.q4_project([o_job], o, H * v, n, [y])
        rt.synchronize()
        check_rotated(q, before[0], positions, freq, factor, nope, True)
        check_rotated(kv[:, None], before[1][:, None], positions, freq, factor, rank, True)
        plain = o.reshape(n, H * v).double() @ o_plain.T
        # Weights in 4 bits are exact; a sum of bf16 products, then half a bf16 step.
        size = o.reshape(n, H * v).double().abs() @ o_plain.abs().T
        assert ((y.double() - plain).abs() <= plain.abs() * HALF + size * 2.0 ** -11).all()
        return q, o

    first, second = rt.create_latent_kv(rank, rope), rt.create_latent_kv(rank, rope)
    x = bf16(g, rows, E, std=0.3)
    at = torch.arange(rows, dtype=torch.int32, device=torch_dev)
    q, o = layer(x, at, lambda q, kv, o: rt.latent_attention_prefill(weights, first, q, kv, norm, EPS, rows, o))
    ref, bound = attention(q, *held(first), kv_b, nope, scale, 0)
    assert_attention(o, ref, bound, "prompt")
    for step in range(3):
        at = torch.tensor([rows + step, step], dtype=torch.int32, device=torch_dev)
        q, o = layer(bf16(g, 2, E, std=0.3), at,
                     lambda q, kv, o: rt.latent_attention(weights, [first, second], q, kv, norm, EPS, o))
        for b, (cache, start) in enumerate(((first, rows + step), (second, step))):
            assert cache.sequence_length == start + 1
            ref, bound = attention(q[b:b + 1], *held(cache), kv_b, nope, scale, start)
            assert_attention(o[b:b + 1], ref, bound, f"step {step} of sequence {b}")
    for c in (first, second):
        c.close()
