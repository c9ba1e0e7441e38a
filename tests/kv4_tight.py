"""What decode attention over a 4-bit cache of at most 32 tokens may be off by, apart from
the rounding of its outputs."""
from __future__ import annotations

import math

import torch

from kv4_util import GROUP, held, spread


def decode_bound(q, kparts, vparts, first):
    """(o, bound) of q [M][H][D] over parts (codes, s, m) [T][KVH][...], row i seeing tokens 0
    .. first + i, T <= 32: one pair of pages, one step of one wave.

    Scores: an fp32 sum of D products of bf16 queries and codes + 136 <= 143 against 136
    sums of the queries, in at most 2 D / 32 + 3 matrix instructions and additions of at
    most 6 roundings each; then a product and three sums: 2^-24 each, of at most
    sum |q| (143 s + 2 |m|).
    Weights: that, two roundings of the exponential, of the reference and of their product
    with s (2^-22 in all), and as bf16 hi + lo 2^-17.
    Outputs: two matrix instructions of codes + 136 <= 143 and two that take 136 off, and the
    offsets' sum: at most 25 roundings of at most sum p (143 s + |m|); the division 2^-23."""
    k, v = (held(*p) for p in (kparts, vparts))
    M, H, D = q.shape
    KVH = k.shape[1]
    qd = q.double()
    ks, km, vs, vm = (spread(p[i].double().abs(), D) for p in (kparts, vparts) for i in (1, 2))
    o, bound = torch.empty_like(qd), torch.empty_like(qd)
    seen = torch.arange(k.shape[0], device=q.device) <= torch.arange(M, device=q.device)[:, None] + first
    for h in range(H):
        g = h // (H // KVH)
        score = qd[:, h] @ k[:, g].T / math.sqrt(D)
        p = torch.softmax(torch.where(seen, score, -math.inf), 1)
        steps = 6 * (2 * -(-D // 32) + 3) + 4
        off = qd[:, h].abs() @ (143 * ks[:, g] + 2 * km[:, g]).T / math.sqrt(D) * steps * 2 ** -24
        off = torch.where(seen, off, 0.0).amax(1, keepdim=True)
        size = p @ (vparts[0][:, g].double().abs() * vs[:, g] + vm[:, g])
        o[:, h] = p @ v[:, g]
        # (A score's error moves its weight and the sum of weights.)
        bound[:, h] = size * (2 * off + 2 ** -17 + 2 ** -21) + p @ (143 * vs[:, g] + vm[:, g]) * 25 * 2 ** -24
    return o, bound


def beyond(o, want, bound):
    """How often bf16 outputs are further off than the bound and their own rounding."""
    err = (o.double() - want).abs()
    return int((~(err <= bound + (want.abs() + bound) * 2 ** -8)).sum())


__all__ = ["GROUP", "beyond", "decode_bound"]
