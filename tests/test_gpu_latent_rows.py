"""GPU tests of latent attention, every row of every head within the bound of what the
form that computes it may round (latent_util.attention_rows)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import qm38
from gpu_util import to_dev, tuned
from latent_util import HALF, assert_attention_rows, attention_rows, rotated, frequencies
from qm38 import synth
from test_gpu_latent import EPS, FORMS, ODD, SMALL, TINY, WIDE, bf16, filled, generator, held, make_weights

pytestmark = pytest.mark.gpu


def check_prefill(rt, form, widths, H, cached, rows, seed, q_std=1.5):
    rank, rope, nope, v = widths
    g = generator(seed)
    kv_b, scale, weights = make_weights(rt, g, H, widths)
    norm = torch.rand(rank, generator=g, device="cuda:0") + 0.5
    cache = filled(rt, g, widths, cached, norm)
    q, kv = bf16(g, rows, H, nope + rope, std=q_std), bf16(g, rows, rank + rope)
    o = torch.full((rows, H, v), float("nan"), dtype=torch.bfloat16, device="cuda:0")
    rt.latent_attention_prefill(weights, cache, q, kv, norm, EPS, rows, o)
    ref, bounds = attention_rows(q, *held(cache), kv_b, nope, scale, cached, form)
    assert_attention_rows(o, ref, bounds, f"{rows} rows on {cached}")
    weights.close()
    cache.close()


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
        ref, bounds = attention_rows(q[b:b + 1], *held(cache), kv_b, nope, scale, lengths[b], "absorbed")
        assert_attention_rows(o[b:b + 1], ref, bounds, f"sequence {b} of {lengths[b]}")
        cache.close()
    weights.close()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("widths", [WIDE, SMALL, ODD, TINY, (200, 8, 128, 40), (512, 64, 64, 128), (128, 64, 128, 64)])
@pytest.mark.parametrize("H,cached,rows", [(1, 0, 1), (5, 0, 33), (3, 1000, 7), (20, 31, 130), (33, 64, 65)])
def test_prompt_widths(torch_dev, form, widths, H, cached, rows):
    with tuned(**FORMS[form]) as rt:
        check_prefill(rt, form.replace("head by head", "expanded"), widths, H, cached, rows, H + rows)


@pytest.mark.parametrize("form,widths,H,cached,rows", [
    # Workgroups of eight waves, from one end of the prompt and from both, and of four.
    *(("expanded", w, *size) for w in (WIDE, SMALL)
      for size in ((130, 20, 300), (66, 1, 520), (130, 7, 250), (20, 333, 300), (1, 0, 1025), (64, 0, 300), (8, 4096, 513))),
    # One split, several, and more than eight.
    ("absorbed", SMALL, 20, 3000, 512), ("absorbed", SMALL, 20, 100, 4096), ("absorbed", SMALL, 64, 2500, 24),
    ("absorbed", SMALL, 2, 0, 700), ("absorbed", WIDE, 32, 20001, 5), ("absorbed", WIDE, 128, 100, 40),
    ("absorbed", TINY, 1024, 5, 70), ("expanded", TINY, 1024, 5, 70),
])
def test_prompt_sizes(torch_dev, form, widths, H, cached, rows):
    with tuned(**FORMS[form]) as rt:
        check_prefill(rt, form, widths, H, cached, rows, H + rows)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("q_std", [0.01, 6.0, 60.0])
def test_prompt_of_flat_and_peaked_scores(torch_dev, form, q_std):
    with tuned(**FORMS[form]) as rt:
        check_prefill(rt, form.replace("head by head", "expanded"), ODD, 12, 700, 300, 2, q_std=q_std)


@pytest.mark.parametrize("widths", [WIDE, SMALL, ODD, TINY, (128, 16, 24, 128), (264, 64, 128, 8)])
@pytest.mark.parametrize("H", [1, 5, 32, 33, 100])
def test_decode_widths(rt, widths, H):
    check_decode(rt, widths, H, [0, 1, 31, 32, 63, 255, 256, 700], H)


@pytest.mark.parametrize("H,lengths", [(128, [4097]), (64, [20000, 3, 8191]), (20, [70001]), (16, [2047, 2048, 2049])])
def test_decode_lengths(rt, H, lengths):
    check_decode(rt, WIDE, H, lengths, H)


def test_decode_of_a_full_batch(rt):
    """64 sequences, the most, of lengths on both sides of blocks, tiles and splits."""
    check_decode(rt, SMALL, 40, [(37 * i * i) % 2500 for i in range(64)], 5)


@pytest.mark.parametrize("q_std", [0.01, 60.0])
def test_decode_of_flat_and_peaked_scores(rt, q_std):
    check_decode(rt, SMALL, 40, [3000, 10], 1, q_std=q_std)


@pytest.mark.parametrize("tiles", [1, 2, 7, 1000])
def test_splits_of_any_size(torch_dev, tiles):
    """Whatever blocks a split takes, one of the last or all of them."""
    with tuned(QM38_LATENT_FORM=1, QM38_LATENT_TILES=tiles) as rt:
        check_decode(rt, SMALL, 40, [1500, 0, 95, 96], 3)
        check_prefill(rt, "absorbed", SMALL, 12, 700, 21, 4)


@pytest.mark.parametrize("form", [*FORMS, "decode"])
def test_a_column_of_weights_above_the_others(torch_dev, form):
    """One latent element's column of W_uk a hundred times the others' sets the step of
    the absorbed queries; the element itself is small in the cache."""
    rank, rope, nope, v = SMALL
    g = generator(81)
    H, rows = 6, 50
    kv_b = bf16(g, H, nope + v, rank, std=rank ** -0.5)
    kv_b[:, :nope, 17] *= 100
    scale = (nope + rope) ** -0.5
    q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
    kv[:, 17] *= 2.0 ** -7
    with tuned(**FORMS.get(form, {})) as rt:
        weights = rt.create_latent_weights(qm38.LatentConfig(H, rank, nope, rope, v, scale), kv_b)
        cache = rt.create_latent_kv(rank, rope)
        o = torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev)
        if form == "decode":
            for i in range(rows):
                rt.latent_attention(weights, [cache], q[i:i + 1].clone(), kv[i:i + 1].clone(), None, 0.0, o[i:i + 1])
        else:
            rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
        kind = "expanded" if form in ("expanded", "head by head") else "absorbed"
        ref, bounds = attention_rows(q, *held(cache), kv_b, nope, scale, 0, kind)
        assert_attention_rows(o, ref, bounds)


@pytest.mark.parametrize("form", FORMS)
def test_q4_weights_as_they_are(torch_dev, form):
    """kv_b as a Q4 job against its own values, whose rounding to bf16 is then half a
    step of each."""
    rank, rope, nope, v = 256, 64, 64, 48
    H, rows = 6, 60
    rng, g = np.random.default_rng(82), generator(82)
    mat = synth.q4_matrix(rng, H * (nope + v), rank)
    dev = tuple(to_dev(a, torch_dev) for a in mat)
    w = synth.unpack_q4(mat[0]).astype(np.float64).reshape(-1, rank // 64, 64)
    w = w * synth.bf16_to_f32(mat[1])[..., None] + synth.bf16_to_f32(mat[2])[..., None]
    kv_b = torch.from_numpy(w.reshape(H, nope + v, rank)).to(torch_dev)
    scale = (nope + rope) ** -0.5
    q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
    with tuned(**FORMS[form]) as rt:
        weights = rt.create_latent_weights(qm38.LatentConfig(H, rank, nope, rope, v, scale),
                                           qm38.Runtime.job(*dev, H * (nope + v)))
        cache = rt.create_latent_kv(rank, rope)
        o = torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev)
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
        ref, bounds = attention_rows(q, *held(cache), kv_b, nope, scale, 0, form.replace("head by head", "expanded"),
                                     weight_step=HALF)
        assert_attention_rows(o, ref, bounds)


def test_every_head_of_a_cache_beyond_32_bit_offsets(rt):
    """7.5 million tokens alike and a hundred others behind them: the softmax over 101
    tokens, one of which counts 7.5 million times."""
    rank, rope, nope, v = WIDE
    g = generator(83)
    H, alike, chunk = 24, 7_500_000, 500_000
    kv_b, scale, weights = make_weights(rt, g, H, WIDE)
    one, others = bf16(g, 1, rank + rope, std=0.01), bf16(g, 100, rank + rope)
    cache, few = rt.create_latent_kv(rank, rope), rt.create_latent_kv(rank, rope)
    cache.reserve(alike + 100)
    many = one.expand(chunk, -1).contiguous()
    for _ in range(alike // chunk):
        cache.append(many, None, 0.0, chunk)
    cache.append(others, None, 0.0, 97)
    few.append(torch.cat([one, others]), None, 0.0, 101)
    count = torch.ones(101, device="cuda:0")
    count[0] = alike
    q = bf16(g, 3, H, nope + rope, std=8.0)
    o = torch.empty(3, H, v, dtype=torch.bfloat16, device="cuda:0")
    rt.latent_attention(weights, [cache], q[:1], others[97:98], None, 0.0, o[:1])
    rt.latent_attention_prefill(weights, cache, q[1:], others[98:], None, 0.0, 2, o[1:])
    # About 256 splits, of 64 tokens an addition.
    ref, bounds = attention_rows(q, *held(few), kv_b, nope, scale, 98, "absorbed", count=count, adds=alike / 256 / 16)
    assert_attention_rows(o, ref, bounds)
    cache.close()
    few.close()
    weights.close()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,width,offset,rd", [(5, 20, 192, 128, 64), (7, 5, 65, 3, 30), (300, 3, 128, 0, 128)])
def test_every_pair_of_rotary_positions(rt, interleaved, rows, heads, width, offset, rd):
    """Each pair within fp32's part of its own elements (2^-20 of |a| + |b|: the angle's
    rounding below pi to 2^-23, sine and cosine to an ulp or two, three roundings) and
    half a bf16 step; the pairs are of sizes from 2^-20 to 2^20."""
    g = generator(84)
    x = bf16(g, rows, heads, width)
    size = torch.randint(-20, 21, (rd // 2,), generator=g, device="cuda:0").double().exp2()
    part = x[..., offset:offset + rd]
    part.mul_((size.repeat_interleave(2) if interleaved else size.repeat(2)).to(torch.bfloat16))
    positions = torch.randint(0, 1 << 31, (rows,), generator=g, device="cuda:0").to(torch.int32)
    freq, factor = frequencies(rd, 1e6, "yarn", 8.0, 4096, device="cuda:0")
    out = torch.full_like(x, 7.0)
    rt.rotary(qm38.RotaryConfig(rd, interleaved, 1e6, "yarn", 8.0, 4096), [(x, out, heads, width, offset)], rows,
              positions=positions)
    ref = rotated(x, positions, freq, factor, offset, interleaved)
    pair = part.double().abs()
    pair = pair.unflatten(-1, (-1, 2)).sum(-1) if interleaved else pair.unflatten(-1, (2, -1)).sum(-2)
    pair = pair.repeat_interleave(2, -1) if interleaved else pair.repeat(1, 1, 2)
    got, ref = out[..., offset:offset + rd].double(), ref[..., offset:offset + rd]
    assert ((got - ref).abs() <= (ref.abs() * HALF + pair * factor * 2.0 ** -20) * (1 + HALF)).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("power", [-10, 10])
def test_parts_of_a_score_of_different_sizes(torch_dev, form, power):
    """Latents 2^power and keys 2^-power of the usual size, the two parts of a query the
    other way round: neither part of a score loses precision."""
    rank, rope, nope, v = SMALL
    g = generator(85)
    H, rows = 6, 200
    with tuned(**FORMS[form]) as rt:
        kv_b, scale, weights = make_weights(rt, g, H, SMALL)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        kv[:, :rank] *= 2.0 ** power
        kv[:, rank:] *= 2.0 ** -power
        q[..., :nope] *= 2.0 ** -power
        q[..., nope:] *= 2.0 ** power
        cache = rt.create_latent_kv(rank, rope)
        o = torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev)
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
        ref, bounds = attention_rows(q, *held(cache), kv_b, nope, scale, 0, form.replace("head by head", "expanded"))
        assert_attention_rows(o, ref, bounds)


@pytest.mark.parametrize("form", FORMS)
def test_tokens_of_different_sizes_in_a_tile(torch_dev, form):
    """A token whose latent is 2^16 times its neighbours', and which rows leave nothing
    (the shared key's part decides), costs no row precision."""
    rank, rope, nope, v = SMALL
    g = generator(86)
    H, rows = 6, 200
    with tuned(**FORMS[form]) as rt:
        kv_b, scale, weights = make_weights(rt, g, H, SMALL)
        q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
        q[..., :nope] = 0
        q[..., nope:] = 1
        kv[[5, 110], :rank] *= 2.0 ** 16
        kv[[5, 110], rank:] = -100.0
        cache = rt.create_latent_kv(rank, rope)
        o = torch.empty(rows, H, v, dtype=torch.bfloat16, device=torch_dev)
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
        ref, bounds = attention_rows(q, *held(cache), kv_b, nope, scale, 0, form.replace("head by head", "expanded"))
        assert_attention_rows(o, ref, bounds)
