"""Plain forms in 64 bits of rotary positions and latent attention, and the
error bounds of the kernels that compute them in fewer bits."""
from __future__ import annotations

import math

import torch

HALF = 2.0 ** -8  # at most half a bf16 step, relative


def rotated(x, positions, freq, factor, offset, interleaved):
    """x [rows][heads][width] in float64, its pairs from `offset` on turned."""
    rd = 2 * len(freq)
    y = x.double().clone()
    angle = positions.double()[:, None, None] * freq
    cos, sin = torch.cos(angle) * factor, torch.sin(angle) * factor
    part = y[..., offset:offset + rd]
    a, b = (part[..., 0::2].clone(), part[..., 1::2].clone()) if interleaved else (
        part[..., :rd // 2].clone(), part[..., rd // 2:].clone())
    if interleaved:
        part[..., 0::2], part[..., 1::2] = a * cos - b * sin, b * cos + a * sin
    else:
        part[..., :rd // 2], part[..., rd // 2:] = a * cos - b * sin, b * cos + a * sin
    return y


def frequencies(rd, theta, scaling="none", factor=1.0, original=0, fast=32.0, slow=1.0, device="cpu"):
    i = torch.arange(rd // 2, dtype=torch.float64, device=device)
    f = theta ** (-2 * i / rd)
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    at = [rd * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (fast, slow)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rd - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1


def quantised(x):
    """(codes float64, scale) of rows x (float64 holding fp32 values): the scale
    and the quotients as fp32 has them."""
    amax = x.abs().amax(-1, keepdim=True).float()
    # (torch multiplies by the reciprocal where the divisor is a Python number.)
    scale = (amax / torch.full_like(amax, 127)).clamp(min=1.1754943508222875e-38)
    t = (x.float() / scale).clamp(-127, 127).double()
    return torch.sign(t) * torch.floor(t.abs() + 0.5), scale


def attention(q, latent, key, kv_b, nope, scale, start):
    """Latent attention in float64: q [M][H][nope + rope], the cache's latents
    and keys [T][...] as it holds them, kv_b [H][nope + v][rank]; row i sees
    tokens 0 .. start + i.  Returns (o [M][H][v], bound of the kernels' error)."""
    q, w = q.double().transpose(0, 1), kv_b.double()  # [H][M][...]
    T, M = latent.shape[0], q.shape[1]
    k = latent @ w[:, :nope].transpose(1, 2)  # [H][T][nope]
    v = latent @ w[:, nope:].transpose(1, 2)
    score = (q[..., :nope] @ k.transpose(1, 2) + q[..., nope:] @ key.T) * scale
    seen = torch.arange(T, device=q.device) <= torch.arange(M, device=q.device)[:, None] + start
    p = torch.softmax(torch.where(seen, score, -math.inf), -1)
    o = p @ v
    # Errors, each rounding at its largest.  Scores: the expanded form rounds its
    # keys (to fp16; half a step of bf16 is allowed); the absorbed one the queries in the latent space to 1 / 65024
    # of their largest element (and the rotated part likewise).
    absorbed = q[..., :nope] @ w[:, :nope]
    a = (q[..., :nope].abs() @ k.abs().transpose(1, 2)) * HALF
    b = absorbed.abs().amax(-1, keepdim=True) / 65024 * latent.abs().sum(-1)
    b = b + q[..., nope:].abs().amax(-1, keepdim=True) / 65024 * key.abs().sum(-1)
    fp32 = (q[..., :nope].abs() @ k.abs().transpose(1, 2) + q[..., nope:].abs() @ key.abs().T) * 1e-5
    ds = torch.where(seen, (torch.maximum(a, b) + fp32) * scale, 0.0).amax(-1, keepdim=True)
    # p is off by a factor of at most e^(2 ds), its rounding and the values'
    # (expanded) or the joined sums' (absorbed: of every latent element, which
    # the products with W_uv add up) by half a step each.
    spread = p @ latent.abs()  # [H][M][rank]
    each = spread @ w[:, nope:].abs().transpose(1, 2)
    bound = each * (torch.expm1(2 * ds) + 2 * HALF) * (1 + 2 * HALF) + o.abs() * HALF
    return o.transpose(0, 1), bound.transpose(0, 1)


def assert_attention(got, ref, bound, what=""):
    """Every output within the bound; and in the norm within 2^-7: a result goes
    through at most four roundings of at most 2^-8 (rms 2^-8 / sqrt 3 each), which
    add up to 1.2 * 2^-8 where they are independent."""
    got = got.double()
    assert torch.isfinite(got).all(), what
    err = (got - ref).abs()
    assert (err <= bound + 1e-30).all(), f"{what}: {float((err / (bound + 1e-30)).max()):.3f} of the bound"
    norm = float((got - ref).norm() / ref.norm())
    assert norm <= 2.0 ** -7, f"{what}: {norm:.2e} off in the norm"
    return norm
