"""GPU tests of latent attention on weights and rows at the ends of their types:
numbers that are none, and scales far from one."""
from __future__ import annotations

import pytest
import torch

import qm38
from gpu_util import tuned
from test_gpu_latent import FORMS, SMALL, bf16, generator

pytestmark = pytest.mark.gpu


def outputs(rt, widths, kv_b, q, kv, decode):
    """All rows as a prompt, or the last one decoded behind the others."""
    rank, rope, nope, v = widths
    rows, H = q.shape[:2]
    weights = rt.create_latent_weights(qm38.LatentConfig(H, rank, nope, rope, v, (nope + rope) ** -0.5), kv_b)
    cache = rt.create_latent_kv(rank, rope)
    o = torch.zeros(rows, H, v, dtype=torch.bfloat16, device="cuda:0")
    if decode:
        cache.append(kv, None, 0.0, rows - 1)
        rt.latent_attention(weights, [cache], q[rows - 1:].clone(), kv[rows - 1:].clone(), None, 0.0, o[rows - 1:])
        o = o[rows - 1:]
    else:
        rt.latent_attention_prefill(weights, cache, q, kv, None, 0.0, rows, o)
    torch.cuda.synchronize()
    weights.close()
    cache.close()
    return o


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("form", [*FORMS, "decode"])
def test_key_weights_that_are_none(torch_dev, form, value):
    """A NaN or an infinity among a head's W_uk is in every score of that head, and
    in nothing of the others."""
    rank, rope, nope, v = SMALL
    g = generator(51)
    H, rows = 5, 40
    kv_b = bf16(g, H, nope + v, rank, std=rank ** -0.5)
    q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
    worse = kv_b.clone()
    worse[3, 7, 200] = value
    with tuned(**FORMS.get(form, {})) as rt:
        o, clean = (outputs(rt, SMALL, w, q, kv, form == "decode") for w in (worse, kv_b))
    assert torch.isnan(o[:, 3]).all()
    others = [0, 1, 2, 4]
    assert torch.isfinite(clean).all() and torch.equal(o[:, others], clean[:, others])


@pytest.mark.parametrize("power", [-80, -60, 64, 80])
@pytest.mark.parametrize("form", [*FORMS, "decode"])
def test_key_weights_of_any_size(torch_dev, form, power):
    """W_uk times 2^power and queries times 2^-power have the same scores, formed
    by the same steps: no bit of the outputs differs."""
    rank, rope, nope, v = SMALL
    g = generator(52)
    H, rows = 5, 40
    kv_b = bf16(g, H, nope + v, rank, std=rank ** -0.5)
    q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
    scaled, scaled_q = kv_b.clone(), q.clone()
    scaled[:, :nope] *= 2.0 ** power
    scaled_q[..., :nope] *= 2.0 ** -power
    with tuned(**FORMS.get(form, {})) as rt:
        o, plain = (outputs(rt, SMALL, w, x, kv, form == "decode") for w, x in ((scaled, scaled_q), (kv_b, q)))
    assert torch.isfinite(plain).all() and torch.equal(o, plain)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("power", [-20, 0, 12])
@pytest.mark.parametrize("form", [*FORMS, "decode"])
def test_value_weights_that_are_none(torch_dev, form, power, value):
    """A NaN or an infinity in a row of W_uv is in that element of the head's outputs;
    the others, at weights of any size, keep every bit."""
    rank, rope, nope, v = SMALL
    g = generator(53)
    H, rows = 5, 40
    kv_b = bf16(g, H, nope + v, rank, std=rank ** -0.5)
    kv_b[:, nope:] *= 2.0 ** power
    q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
    # Not the row that is the head's largest, which the finite ones would lose too.
    element = int(kv_b[3, nope:].double().abs().sum(1).argmin())
    worse = kv_b.clone()
    worse[3, nope + element, 200] = value
    with tuned(**FORMS.get(form, {})) as rt:
        o, clean = (outputs(rt, SMALL, w, q, kv, form == "decode") for w in (worse, kv_b))
    assert torch.isfinite(clean).all()
    assert not torch.isfinite(o[:, 3, element]).any()
    o[:, 3, element] = clean[:, 3, element]
    assert torch.equal(o, clean)


@pytest.mark.parametrize("form", [*FORMS, "decode"])
def test_weights_near_the_largest(torch_dev, form):
    """Weights whose row sums times 127 pass fp32, with cached tokens and queries as
    far below one: what weights near one give, times a power of two."""
    rank, rope, nope, v = SMALL
    g = generator(54)
    H, rows = 5, 40
    kv_b = bf16(g, H, nope + v, rank, std=rank ** -0.5)
    q, kv = bf16(g, rows, H, nope + rope), bf16(g, rows, rank + rope)
    scaled, scaled_q, scaled_kv = kv_b * 2.0 ** 118, q.clone(), kv * 2.0 ** -60
    assert float(scaled.double().abs().sum(2).amin()) * 127 > torch.finfo(torch.float32).max
    scaled_q[..., :nope] *= 2.0 ** -58  # W_uk 2^118, latents 2^-60
    scaled_q[..., nope:] *= 2.0 ** 60   # keys 2^-60
    with tuned(**FORMS.get(form, {})) as rt:
        o = outputs(rt, SMALL, scaled, scaled_q, scaled_kv, form == "decode").double() * 2.0 ** -58
        plain = outputs(rt, SMALL, kv_b, q, kv, form == "decode").double()
    # The same but for the powers under which fp16 holds P and the expanded keys and
    # values, which need not be the same: 2^-11 in each of P and V, of sum p |v|, and
    # about as much of the scores; at most 40 tokens make that sqrt(40) of |o|.  Then
    # two roundings to bf16 of 2^-8: 4 * 6.4 * 2^-11 + 2^-7 < 2^-5.5.
    assert torch.isfinite(plain).all()
    assert ((o - plain).norm(dim=-1) <= 2.0 ** -5.5 * plain.norm(dim=-1)).all()


def test_rows_that_are_none_in_a_batch(rt):
    """Of a batch, the sequences that hold a NaN or an infinity, cached or new, are none
    in every head, a head whose query does in itself alone; the others keep every bit."""
    rank, rope, nope, v = SMALL
    g = generator(55)
    H, cached = 40, 70
    lengths = [cached] * 6
    kv_b = bf16(g, H, nope + v, rank, std=rank ** -0.5)
    weights = rt.create_latent_weights(qm38.LatentConfig(H, rank, nope, rope, v, (nope + rope) ** -0.5), kv_b)
    old, q, kv = bf16(g, cached, rank + rope), bf16(g, 6, H, nope + rope), bf16(g, 6, rank + rope)
    bad_old, bad_q, bad_kv = old.clone(), q.clone(), kv.clone()
    bad_old[31, 5] = float("nan")           # sequence 0: a latent among its tokens,
    bad_old[64, rank + 1] = float("inf")    # and a key
    bad_kv[2, 100] = -float("inf")          # sequence 2: its new latent
    bad_kv[3, rank + 7] = float("nan")      # sequence 3: its new key
    bad_q[4, 33, 9] = float("nan")
    bad_q[5, 2, nope + 1] = float("inf")
    outs = []
    for first, x, rows in ((old, q, kv), (bad_old, bad_q, bad_kv)):
        caches = [rt.create_latent_kv(rank, rope) for _ in lengths]
        for b, cache in enumerate(caches):
            cache.append(first if b == 0 else old, None, 0.0, cached)
        o = torch.zeros(6, H, v, dtype=torch.bfloat16, device="cuda:0")
        rt.latent_attention(weights, caches, x, rows, None, 0.0, o)
        outs.append(o)
        torch.cuda.synchronize()
        for cache in caches:
            cache.close()
    clean, o = outs
    none = torch.zeros(6, H, dtype=torch.bool, device="cuda:0")
    none[[0, 2, 3]] = True
    none[4, 33] = none[5, 2] = True
    assert torch.isfinite(clean).all()
    assert torch.isnan(o[none]).all() and torch.equal(o[~none], clean[~none])
    weights.close()
