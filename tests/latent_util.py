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


FP16 = 2.0 ** -11 * 1.0625  # half an fp16 step, relative, and fp32's errors of what is rounded


def _moved_by_queries(p, k, v, o, q):
    """sqrt(sum_d q_d^2 |sum_t p_t k_td (v_t - o)|^2) for every (head, row): how far
    independent errors of size q_d in the elements of a query move its output."""
    heads, rows, tokens = p.shape
    out = torch.empty(heads, rows, dtype=torch.float64, device=p.device)
    step = max(1, 2 ** 27 // (tokens * k.shape[-1]))
    for h in range(heads):
        for lo in range(0, rows, step):
            w = p[h, lo:lo + step, None] * k[h].T  # [rows][d][T]
            c = w @ v[h] - w.sum(-1, keepdim=True) * o[h, lo:lo + step, None]
            out[h, lo:lo + step] = (q[h, lo:lo + step] ** 2 * (c ** 2).sum(-1)).sum(-1).sqrt()
    return out


def attention_rows(q, latent, key, kv_b, nope, scale, start, form, count=None, adds=None, weight_step=0.0):
    """Latent attention in float64 as attention() gives it, and for every (row, head)
    a bound of the norm over v of what `form`'s roundings may add, and that norm's
    standard deviation: (o [M][H][v], (bound, deviation) [M][H]).

    A rounding's error is at most half a step, h, and has a variance of at most h^2 / 3;
    independent ones are added by their variances, and the bound takes the sum's
    standard deviation five times.  Scores off by d_t move o by
    sum p_t (e^(d_t) - 1) (v_t - o) / sum p_t e^(d_t).
    Expanded: keys to fp16 (independent from token to token), queries to fp16 (the same
    for all tokens).  Absorbed: queries in the latent space to steps of |q_nope| times
    the largest column norm of the head's W_uk / 32512, rotated ones to their largest
    element / 32512 (the same for all tokens: taken as if they always moved o alike).
    weight_step: half a step of weights that were rounded (likewise).
    Sums: P to fp16 (its least parts to 2^-30 of the largest), expanded values to fp16,
    joined sums to two bf16 terms (2^-17), `adds` fp32 additions one behind the other
    (16 tokens each).  Then the output's half bf16 step.
    count: how often each token stands in the cache."""
    q, w = q.double().transpose(0, 1), kv_b.double()  # [H][M][...]
    w_uk, w_uv = w[:, :nope], w[:, nope:]
    T, M = latent.shape[0], q.shape[1]
    qn, qr = q[..., :nope], q[..., nope:]
    k, v = latent @ w_uk.transpose(1, 2), latent @ w_uv.transpose(1, 2)  # [H][T][...]
    score = (qn @ k.transpose(1, 2) + qr @ key.T) * scale
    seen = torch.arange(T, device=q.device) <= torch.arange(M, device=q.device)[:, None] + start
    log_count = torch.zeros(T, dtype=torch.float64, device=q.device) if count is None else torch.log(count.double())
    p = torch.softmax(torch.where(seen, score + log_count, -math.inf), -1)
    o = p @ v
    size_v = v.norm(dim=-1)[:, None]  # [H][1][T]
    apart = (size_v ** 2 - 2 * o @ v.transpose(1, 2) + (o ** 2).sum(-1, keepdim=True)).clamp(min=0).sqrt()

    half = FP16 / math.sqrt(3)
    each = torch.zeros_like(score)  # variances of errors of a token's own, of those of all tokens
    alike = torch.zeros_like(score)
    parts = []  # standard deviations of o's errors
    if form == "expanded":
        each = half ** 2 * (qn ** 2 @ (k ** 2).transpose(1, 2) + qr ** 2 @ (key ** 2).T)
        both = torch.cat((k, key.expand(len(k), -1, -1)), -1)
        parts.append(scale * half * _moved_by_queries(p, both, v, o, q))
        size = qn.abs() @ k.abs().transpose(1, 2) + qr.abs() @ key.abs().T
    else:
        step = qn.norm(dim=-1, keepdim=True) * w_uk.norm(dim=1).amax(-1)[:, None, None] * 1.0002 / 32512
        step_key = qr.abs().amax(-1, keepdim=True) / 32512
        alike = (step ** 2 * (latent ** 2).sum(-1) + step_key ** 2 * (key ** 2).sum(-1)) / 12
        size = (qn @ w_uk).abs() @ latent.abs().T + qr.abs() @ key.abs().T
    if weight_step:
        alike = alike + weight_step ** 2 / 3 * (qn ** 2 @ (w_uk ** 2) @ (latent ** 2).T)
    # fp32: sums of up to 128 products, 2^-24 sqrt(128) of the magnitudes; the exponent's few roundings.
    fp32 = 2.0 ** -20 * scale * size + 2.0 ** -22 * score.abs()
    each, alike = scale * each.sqrt(), scale * alike.sqrt()
    total = (p * torch.expm1(5 * (2 * each ** 2 + alike ** 2).sqrt() + fp32)).sum(-1)
    assert (total < 0.5).all(), "scores too uncertain for a test"
    parts.append(((p * torch.expm1(5 * each) / 5 * apart) ** 2).sum(-1).sqrt())
    parts.append((p * torch.expm1(5 * alike) / 5 * apart).sum(-1))
    parts = [part / (1 - total) for part in parts]

    rounded = 2 if form == "expanded" else 1  # P, and expanded values
    parts.append(half * math.sqrt(rounded) * ((p * size_v) ** 2).sum(-1).sqrt())
    x = p @ latent  # [H][M][rank]
    spread = (x ** 2 @ (w_uv ** 2).transpose(1, 2)).sum(-1).sqrt()
    parts.append(((2.0 ** -17 if form == "absorbed" else 0.0) + weight_step) / math.sqrt(3) * spread)
    small = (p * torch.expm1(fp32) * apart).sum(-1) / (1 - total)  # fp32's part, and P's least
    small = small + (p * size_v).sum(-1) * (T / 16 if adds is None else adds) * 2.0 ** -24
    small = small + 2.0 ** -30 * torch.where(seen, size_v, 0.0).sum(-1)
    small = small + 2.0 ** -20 * (x.abs() @ w_uv.abs().transpose(1, 2)).norm(dim=-1)
    size_o = o.norm(dim=-1)
    bound = (5 * sum(parts) + small) * (1 + HALF) + HALF * size_o
    # Over many values a step's square is 0.54 of its value's at the bottom of a binade.
    deviation = (0.6 * (sum(part ** 2 for part in parts) + HALF ** 2 / 3 * size_o ** 2)).sqrt() + small
    return o.transpose(0, 1), (bound.T, deviation.T)


def assert_attention_rows(got, ref, bounds, what=""):
    """Every row of every head within its own bound; and 64 or more of them together
    within their standard deviation.  That is one of many values: the squares of errors
    that are uniform in +-h have the mean h^2 / 3 and the deviation 0.9 of that, and the
    sum of n alike ones is within 5 * 0.9 / sqrt(n) of its mean; of values x of different
    sizes n is (sum x^2)^2 / sum x^4."""
    got, (bound, deviation) = got.double(), bounds
    assert torch.isfinite(got).all(), what
    err = (got - ref).norm(dim=-1)
    part = err / (bound + 1e-30)
    row, head = divmod(part.flatten().argmax().item(), err.shape[1])
    assert (part <= 1).all(), (f"{what}: row {row}, head {head}: {float(err[row, head]):.3e} off of "
                               f"{float(ref[row, head].norm()):.3e}, bound {float(bound[row, head]):.3e}")
    n = float((ref ** 2).sum() ** 2 / ((ref ** 4).sum() + 1e-300))
    together = float(err.norm() / (deviation.norm() + 1e-30)) / math.sqrt(1 + 4.5 / math.sqrt(n + 1e-30))
    assert err.numel() < 64 or together <= 1, f"{what}: {together:.3f} standard deviations off together"
    return float(part.max()), together
