"""Plain forms of the 4-bit KV cache and of attention over what a cache holds,
and the error bounds of the kernels."""
from __future__ import annotations

import math

import torch

from latent_util import HALF, frequencies, rotated

GROUP = 64
FLT_MIN = 1.1754943508222875e-38


def bf16_bits(t):
    return t.to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xFFFF


def quantised(x):
    """(codes int8 [...][D], scales and offsets bf16 [...][groups]) of fp32 rows, as fp32 has them."""
    codes, scales, offsets = [], [], []
    for part in x.split(GROUP, -1):
        low, high = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
        half = high * 0.5 - low * 0.5
        # (torch multiplies by the reciprocal where the divisor is a Python number.)
        s = (half / torch.full_like(half, 7.5)).clamp(min=FLT_MIN).to(torch.bfloat16)
        m = (low + s.float() * 8).to(torch.bfloat16)
        c = torch.round(((part - m.float()) / s.float()).clamp(-8, 7))
        bad = ~torch.isfinite(part).all(-1, keepdim=True)
        nan = torch.full_like(s, math.nan)
        codes.append(torch.where(bad, torch.zeros_like(c), c).to(torch.int8))
        scales.append(torch.where(bad, nan, s))
        offsets.append(torch.where(bad, nan, m))
    return torch.cat(codes, -1), torch.cat(scales, -1), torch.cat(offsets, -1)


def quantised8(x):
    """(codes int8 [...][D], scale fp32 [...][1]) of the 8-bit cache."""
    top = x.abs().amax(-1, keepdim=True)
    s = (top / torch.full_like(top, 127)).clamp(min=FLT_MIN)
    t = (x / s).clamp(-127, 127).double()
    return (torch.sign(t) * torch.floor(t.abs() + 0.5)).to(torch.int8), s


def spread(per_group, D):
    """[...][groups] -> [...][D]"""
    return per_group.repeat_interleave(GROUP, -1)[..., :D]


def held(codes, s, m):
    """What 4-bit codes stand for, in float64."""
    D = codes.shape[-1]
    return codes.double() * spread(s.double(), D) + spread(m.double(), D)


def read(cache, device="cuda:0"):
    """A cache's content as tensors: ((codes, s, m) of K, of V), s and m bf16, or
    ((codes, scale) of K, of V) of an 8-bit one."""
    k, v, ks, vs = (torch.from_numpy(a).to(device) for a in cache_arrays(cache))
    if cache.bits == 8:
        return (k, ks[..., None]), (v, vs[..., None])
    out = []
    for c, w in ((k, ks), (v, vs)):
        w = w.view(torch.bfloat16)
        out.append((c, w[..., 0].contiguous(), w[..., 1].contiguous()))
    return tuple(out)


def cache_arrays(cache):
    return [a.view("int16") if a.dtype == "uint16" else a for a in cache.read()]


def values(cache):
    """Keys and values of a cache [T][KVH][D] and what bounds their parts, in float64."""
    out = []
    for part in read(cache):
        if cache.bits == 8:
            x = part[0].double() * part[1].double()
            out.append((x, x.abs()))
        else:
            c, s, m = part
            D = c.shape[-1]
            out.append((held(c, s, m), c.double().abs() * spread(s.double(), D) + spread(m.double().abs(), D)))
    return out


def attention(q, gate, kv, first):
    """q [M][H][D] over a cache's values() in float64, row i seeing tokens 0 .. first + i;
    returns (o, bound of a kernel's error before its last rounding).

    Scores are fp32 sums of D exact products (a chain of D / 32 matrix instructions,
    each a tree: 2^-16 of the sum of magnitudes covers it); a weight's relative error
    is that and two roundings of the exponential; weights and values round to fp16
    at most once each in the products (2^-11 each), or less."""
    (k, ka), (v, va) = kv
    M, H, D = q.shape
    KVH = k.shape[1]
    qd = q.double()
    o, bound = torch.empty_like(qd), torch.empty_like(qd)
    seen = torch.arange(k.shape[0], device=q.device) <= torch.arange(M, device=q.device)[:, None] + first
    for h in range(H):
        g = h // (H // KVH)
        score = qd[:, h] @ k[:, g].T / math.sqrt(D)
        size = torch.where(seen, qd[:, h].abs() @ ka[:, g].T / math.sqrt(D), 0.0).amax(1)
        p = torch.softmax(torch.where(seen, score, -math.inf), 1)
        o[:, h] = p @ v[:, g]
        bound[:, h] = (p @ va[:, g]) * (2 ** -10 + 2 * (size * 2 ** -16 + 2 ** -20))[:, None]
    if gate is not None:
        sig = torch.sigmoid(gate.double())
        o, bound = o * sig, bound * sig + o.abs() * sig * 2 ** -20
    return o, bound


def check(o, want, bound):
    """bf16 outputs o within the bound and the last rounding."""
    err = (o.double() - want).abs()
    assert torch.isfinite(o).all()
    bad = err > bound + (want.abs() + bound) * HALF
    assert not bad.any(), (int(bad.sum()), float((err / (bound + want.abs() * HALF + 1e-300)).max()))


__all__ = ["attention", "check", "frequencies", "held", "quantised", "quantised8", "read", "rotated", "spread", "values"]
