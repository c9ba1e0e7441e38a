"""Latent attention and what it needs, as cases that can be timed and checked.

In latent attention the keys and values of all heads come from one vector per
token, c_t (rank elements, RMS-normalised), and one rotated key k_t (rope
elements) that the heads share.  With W_uk [head][nope][rank] and W_uv
[head][v][rank] the rows of one projection `kv_b` [head][nope + v][rank],

  score(i, t, h) = scale * (q_nope[i, h] . W_uk[h] c_t + q_rope[i, h] . k_t)
  o[i, h]        = sum_t softmax_t(score)[t] * W_uv[h] c_t

The cache holds c_t and k_t in 8 bits, each with one fp32 scale per token:
s = max(absmax / 127, FLT_MIN), code = round half away(clamp(x / s, -127, 127)).

Four kinds, each one pass through the public entry points of qm38.Runtime:

  rotary   rotary positions on part of every head, out of place     rotary
  cache    rows normalised and quantised behind a cached prefix,    LatentKv.append, LatentKv.load
           then the new rows read back
  decode   one new token for each sequence of a ragged batch        latent_attention
  prefill  new rows of one sequence over its cached prefix          latent_attention_prefill

A pass can be repeated on its state: the caches go back to their cached length
first, as in a program that drops draft tokens.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
FLT_MIN = 1.1754943508222875e-38
THETA = 1e6

# (rank, rope, nope, v): the usual widths of latent attention, a small model's,
# and one whose widths fill no tile.
WIDE, SMALL, ODD = (512, 64, 128, 128), (256, 32, 64, 64), (384, 48, 96, 80)


def _widths(widths):
    return dict(zip(("rank", "rope", "nope", "v"), widths))


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # A decode batch's rotation: the launch and its latency count.
        dict(name="rotary_5", kind="rotary", rows=5, heads=20, interleaved=True, scaling="yarn", factor=8.0, **_widths(WIDE)),
        # A prompt chunk's, half layout, positions scaled for a longer context.
        dict(name="rotary_2048", kind="rotary", rows=2048, heads=64, interleaved=False, scaling="yarn", factor=4.0, **_widths(WIDE)),
        # A decode batch's tokens of one program that checks its cache.
        dict(name="cache_33", kind="cache", rows=33, cached=1000, **_widths(SMALL)),
        # A long prompt's chunk into the cache.
        dict(name="cache_8192", kind="cache", rows=8192, cached=4001, **_widths(WIDE)),
        # One young request of a small model: latency.
        dict(name="decode_1_small", kind="decode", heads=8, lengths="500", **_widths(SMALL)),
        # One request of a large model's share of heads at a long context.
        dict(name="decode_32k", kind="decode", heads=32, lengths="32768", **_widths(WIDE)),
        # All heads at a long context: the products bound it.
        dict(name="decode_128k", kind="decode", heads=128, lengths="131071", **_widths(WIDE)),
        # Requests of very different ages in one batch, one of them new.
        dict(name="decode_ragged", kind="decode", heads=64, lengths="4096,32768,20001,777,65535,16000,0,8191", **_widths(WIDE)),
        # Verification of a few drafted tokens at a long context.
        dict(name="prefill_5_on_20001", kind="prefill", heads=32, rows=5, cached=20001, **_widths(WIDE)),
        # A short prompt, no size a multiple of a tile's.
        dict(name="prefill_333", kind="prefill", heads=20, rows=333, cached=0, **_widths(ODD)),
        # A prompt's first chunk.
        dict(name="prefill_1024", kind="prefill", heads=64, rows=1024, cached=0, **_widths(WIDE)),
        # A prompt's second chunk with all heads.
        dict(name="prefill_2048_on_4096", kind="prefill", heads=128, rows=2048, cached=4096, **_widths(WIDE)),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "cache", "decode", "decode", "prefill", "prefill"])
    widths = _widths(rng.choice([WIDE, WIDE, SMALL, ODD]))
    heads = rng.choice([5, 8, 20, 32, 64, 100, 128])
    if kind == "rotary":
        return dict(kind=kind, rows=_log_int(rng, 1, 2048), heads=heads, interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "yarn"]), factor=float(rng.choice([2, 4, 32])), **widths)
    if kind == "cache":
        return dict(kind=kind, rows=_log_int(rng, 1, 8192), cached=_log_int(rng, 1, 16384) - 1, **widths)
    if kind == "decode":
        lengths = [_log_int(rng, 1, 65536) - 1 for _ in range(rng.randint(1, 9))]
        return dict(kind=kind, heads=heads, lengths=",".join(map(str, lengths)), **widths)
    rows = _log_int(rng, 2, 2048)
    # No more than the listed long prompt's products.
    cached = min(_log_int(rng, 1, 32768) - 1, int(1.3e9 / (heads * rows)) - rows // 2)
    return dict(kind=kind, heads=heads, rows=rows, cached=max(0, cached), **widths)


# ---------------------------------------------------------------------------
# Inputs, made from the seed alone
# ---------------------------------------------------------------------------
class _Maker:
    """Draws of one seed, in a fixed order."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV)
        self.gen.manual_seed(seed)

    def bf16(self, *shape, std=1.0):
        return (torch.randn(shape, generator=self.gen, device=DEV) * std).to(torch.bfloat16)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.gen, device=DEV) * (hi - lo) + lo

    def positions(self, rows):
        return torch.randint(0, 131072, (rows,), generator=self.gen, device=DEV, dtype=torch.int32)


def _inputs(case, seed):
    """What both sides and exact() start from."""
    mk = _Maker(seed)
    rank, rope = case["rank"], case["rope"]
    s = dict(case=case)
    if case["kind"] == "rotary":
        s["q"] = mk.bf16(case["rows"], case["heads"], case["nope"] + rope)
        s["kv"] = mk.bf16(case["rows"], rank + rope)
        s["positions"] = mk.positions(case["rows"])
        return s
    s["norm"] = mk.uniform(0.5, 1.5, rank)
    if case["kind"] == "decode":
        lengths = [int(n) for n in case["lengths"].split(",")]
        new = len(lengths)
    else:
        lengths, new = [case["cached"]], case["rows"]
    s["lengths"] = lengths
    # The projection's rows (latent and key part, rotated already): of the
    # cached tokens, and of the new ones.
    s["cached"] = [mk.bf16(n, rank + rope) for n in lengths]
    s["kv"] = mk.bf16(new, rank + rope)
    if case["kind"] != "cache":
        s["kv_b"] = mk.bf16(case["heads"], case["nope"] + case["v"], rank, std=rank ** -0.5)
        s["q"] = mk.bf16(new, case["heads"], case["nope"] + rope, std=1.5)
    return s


def _scale(case):
    return (case["nope"] + case["rope"]) ** -0.5


_RT = None


def _library():
    """The package and one runtime for the program, on torch's stream."""
    global _RT
    path = str(Path(__file__).resolve().parents[1] / "qwen38-metal_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qm38
    if _RT is None:
        _RT = qm38.Runtime(0)
    _RT.set_stream(torch.cuda.current_stream())
    return qm38, _RT


def prepare(case, seed):
    s = _inputs(case, seed)
    kind, rank, rope = case["kind"], case["rank"], case["rope"]
    if own:
        qm38, rt = _library()
        s["rt"] = rt
        if kind == "rotary":
            s["config"] = qm38.RotaryConfig(
                rotary_dim=rope, interleaved=case["interleaved"], theta=THETA, scaling=case["scaling"],
                factor=case["factor"], original_positions=16384)
            s["q_out"], s["kv_out"] = torch.empty_like(s["q"]), torch.empty_like(s["kv"])
            return s
        s["caches"] = []
        for rows in s["cached"]:
            cache = rt.create_latent_kv(rank, rope)
            cache.reserve(len(rows) + len(s["kv"]))
            if len(rows):
                cache.append(rows, s["norm"], EPS, len(rows))
            s["caches"].append(cache)
        if kind == "cache":
            s["read"] = torch.empty_like(s["kv"])
            return s
        s["weights"] = rt.create_latent_weights(
            qm38.LatentConfig(case["heads"], rank, case["nope"], rope, case["v"], _scale(case)), s["kv_b"])
        s["o"] = torch.empty(len(s["kv"]), case["heads"], case["v"], dtype=torch.bfloat16, device=DEV)
        return s
    if kind == "rotary":
        return s
    # One padded cache for the batch, with room for the new rows.
    room = max(s["lengths"]) + (1 if kind == "decode" else len(s["kv"]))
    s["codes"] = torch.zeros(len(s["lengths"]), room, rank + rope, dtype=torch.int8, device=DEV)
    s["scales"] = torch.zeros(len(s["lengths"]), room, 2, device=DEV)
    for b, rows in enumerate(s["cached"]):
        s["codes"][b, :len(rows)], s["scales"][b, :len(rows)] = _quantised(rows, s["norm"], rank)
    s["length"] = torch.tensor(s["lengths"], device=DEV)
    return s


# ---------------------------------------------------------------------------
# The plain forms, in 32 bits
# ---------------------------------------------------------------------------
def _frequencies(case):
    """Turns per position of every frequency, and the factor of sine and cosine, in 64 bits."""
    rope = case["rope"]
    i = torch.arange(rope // 2, dtype=torch.float64, device=DEV)
    freq = THETA ** (-2 * i / rope)
    if case["scaling"] == "linear":
        return freq / case["factor"], 1.0
    if case["scaling"] == "yarn":
        # Frequencies that turn often within the original context stay, slow
        # ones are divided by the factor, a ramp between them.
        low, high = (rope * math.log(16384 / (turns * 2 * math.pi)) / (2 * math.log(THETA)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rope - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return freq / case["factor"] * ramp + freq * (1 - ramp), 0.1 * math.log(case["factor"]) + 1.0
    return freq, 1.0


def _plain_rotary(s):
    case, rope = s["case"], s["case"]["rope"]
    freq, factor = _frequencies(case)
    angle = s["positions"].double()[:, None, None] * freq
    cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()

    def turned(x):  # [rows][heads][width], its last `rope` elements rotated
        head, part = x[..., :-rope], x[..., -rope:].float()
        if case["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = part[..., :rope // 2], part[..., rope // 2:]
            part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((head, part.to(torch.bfloat16)), -1)

    return turned(s["q"]), turned(s["kv"][:, None])[:, 0]


def _codes(x):
    top = x.abs().amax(-1, keepdim=True)
    scale = (top / torch.full_like(top, 127)).clamp(min=FLT_MIN)  # (by a number torch multiplies with its reciprocal)
    t = (x / scale).clamp(-127, 127).double()  # adding a half in 32 bits would round up what is just below it
    return (torch.sign(t) * torch.floor(t.abs() + 0.5)).to(torch.int8), scale


def _quantised(rows, norm, rank):
    x = rows.float()
    latent = x[:, :rank]
    latent = latent * torch.rsqrt((latent * latent).mean(-1, keepdim=True) + EPS) * norm
    (c, cs), (k, ks) = _codes(latent), _codes(x[:, rank:])
    return torch.cat((c, k), -1), torch.cat((cs, ks), -1)


def _read(codes, scales, rank):
    x = codes.float()
    return x[..., :rank] * scales[..., :1], x[..., rank:] * scales[..., 1:]


def _plain_append(s):
    """The new rows' codes behind every sequence's cached ones."""
    codes, scales = _quantised(s["kv"], s["norm"], s["case"]["rank"])
    new = torch.arange(len(codes), device=DEV)
    if s["case"]["kind"] == "decode":
        s["codes"][new, s["length"]], s["scales"][new, s["length"]] = codes, scales
    else:
        s["codes"][0, s["length"] + new], s["scales"][0, s["length"] + new] = codes, scales


def _softmax(x):
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_decode(s):
    case = s["case"]
    nope = case["nope"]
    _plain_append(s)
    latent, key = _read(s["codes"], s["scales"], case["rank"])  # [B][T][...]
    w, q = s["kv_b"].float(), s["q"].float()
    absorbed = torch.matmul(q[..., :nope].transpose(0, 1), w[:, :nope]).transpose(0, 1)  # [B][H][rank]
    score = torch.matmul(absorbed, latent.transpose(1, 2)) + torch.matmul(q[..., nope:], key.transpose(1, 2))
    hidden = torch.arange(latent.shape[1], device=DEV) > s["length"][:, None]
    p = _softmax((score * _scale(case)).masked_fill(hidden[:, None], -math.inf))
    mixed = torch.matmul(p, latent).transpose(0, 1)  # [H][B][rank]
    return torch.matmul(mixed, w[:, nope:].transpose(1, 2)).transpose(0, 1).to(torch.bfloat16)


def _plain_prefill(s):
    case = s["case"]
    nope, rows = case["nope"], case["rows"]
    _plain_append(s)
    latent, key = _read(s["codes"][0], s["scales"][0], case["rank"])
    w, q = s["kv_b"].float(), s["q"].float().transpose(0, 1)  # q [H][M][...]
    expanded = torch.matmul(latent, w.transpose(1, 2))  # [H][T][nope + v]
    score = torch.matmul(q[..., :nope], expanded[..., :nope].transpose(1, 2)) + torch.matmul(q[..., nope:], key.T)
    new = torch.arange(rows, device=DEV)[:, None] + s["length"]
    hidden = torch.arange(latent.shape[0], device=DEV) > new
    p = _softmax((score * _scale(case)).masked_fill(hidden, -math.inf))
    return torch.matmul(p, expanded[..., nope:]).transpose(0, 1).to(torch.bfloat16)


def _plain_cache(s):
    _plain_append(s)
    at = s["lengths"][0]
    rank = s["case"]["rank"]
    return torch.cat(_read(s["codes"][0, at:], s["scales"][0, at:], rank), -1).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"rotary": _plain_rotary, "cache": _plain_cache, "decode": _plain_decode, "prefill": _plain_prefill}[kind](s)
    rt, rope = s["rt"], case["rope"]
    if kind == "rotary":
        q, kv = s["q"], s["kv"]
        rt.rotary(s["config"], [(q, s["q_out"], case["heads"], q.shape[2], case["nope"]),
                                (kv, s["kv_out"], 1, kv.shape[1], case["rank"])],
                  case["rows"], positions=s["positions"])
        return s["q_out"], s["kv_out"]
    for cache, length in zip(s["caches"], s["lengths"]):
        cache.truncate(length)
    if kind == "cache":
        cache = s["caches"][0]
        cache.append(s["kv"], s["norm"], EPS, case["rows"])
        cache.load(case["cached"], case["rows"], s["read"])
        return s["read"]
    if kind == "decode":
        rt.latent_attention(s["weights"], s["caches"], s["q"], s["kv"], s["norm"], EPS, s["o"])
    else:
        rt.latent_attention_prefill(s["weights"], s["caches"][0], s["q"], s["kv"], s["norm"], EPS, case["rows"], s["o"])
    return s["o"]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, rank, rope, nope, v = (case[k] for k in ("kind", "rank", "rope", "nope", "v"))
    row, held = 2 * (rank + rope), rank + rope + 8  # bytes of a row given, and of one in the cache
    if kind == "rotary":
        rows, width = case["rows"], case["heads"] * (nope + rope) + rank + rope
        return {"bytes": rows * (4 * width + 4), "flops": 3 * rows * (case["heads"] + 1) * rope}
    if kind == "cache":
        # Rows in, codes out; codes in, rows out.
        return {"bytes": case["rows"] * 2 * (row + held) + 4 * rank, "flops": 8 * case["rows"] * rank}
    heads = case["heads"]
    if kind == "decode":
        new, cached = len(case["lengths"].split(",")), sum(int(n) for n in case["lengths"].split(","))
        seen = cached + new  # (row, visible token) pairs
    else:
        new, cached = case["rows"], case["cached"]
        seen = new * cached + new * (new + 1) // 2
    # The cheaper of the two forms: every row's queries and sums through the
    # latent space, or every token's keys and values out of it.
    absorbed = 2 * heads * (seen * (2 * rank + rope) + new * rank * (nope + v))
    expanded = 2 * heads * (seen * (nope + rope + v) + (cached + new) * rank * (nope + v))
    return {"bytes": cached * held + new * (row + held) + 2 * heads * (nope + v) * rank + 2 * new * heads * (nope + rope + v),
            "flops": min(absorbed, expanded)}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_held(rows, norm, rank):
    """What the cache stands for after these rows: latents and keys."""
    out = []
    for part in (rows[:, :rank].double(), rows[:, rank:].double()):
        if not out:
            part = part / (part.pow(2).sum(1, keepdim=True) / rank + EPS).sqrt() * norm.double()
        step = torch.clamp(part.abs().max(1, keepdim=True).values / 127.0, min=FLT_MIN)
        t = part / step
        out.append(torch.where(t < 0, torch.ceil(t - 0.5), torch.floor(t + 0.5)) * step)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    rank, rope, nope = case["rank"], case["rope"], case["nope"]
    if case["kind"] == "rotary":
        freq, factor = _frequencies(case)
        turn = torch.polar(torch.full((), factor, dtype=torch.float64, device=DEV).expand(case["rows"], rope // 2),
                           s["positions"].double()[:, None] * freq)[:, None]
        out = []
        for x in (s["q"], s["kv"][:, None]):
            x = x.double()
            part = x[..., -rope:]
            pair = part.unflatten(-1, (-1, 2)) if case["interleaved"] else part.unflatten(-1, (2, -1)).transpose(-1, -2)
            pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
            part = (pair if case["interleaved"] else pair.transpose(-1, -2)).flatten(-2)
            out.append(torch.cat((x[..., :-rope], part), -1))
        return out[0], out[1][:, 0]
    if case["kind"] == "cache":
        return torch.cat(_exact_held(s["kv"], s["norm"], rank), 1)
    decode = case["kind"] == "decode"
    o = torch.empty(len(s["kv"]), case["heads"], case["v"], dtype=torch.float64, device=DEV)
    w, q = s["kv_b"].double(), s["q"].double()
    for b, cached in enumerate(s["cached"]):
        rows = slice(b, b + 1) if decode else slice(0, len(s["kv"]))
        latent, key = _exact_held(torch.cat((cached, s["kv"][rows])), s["norm"], rank)
        m, total = q[rows].shape[0], latent.shape[0]
        seen = torch.ones(m, total, dtype=torch.bool, device=DEV).tril(total - m)
        for h in range(case["heads"]):
            if decode:  # keys and values of the head, where the plain form absorbs them
                score = q[rows, h, :nope] @ (latent @ w[h, :nope].T).T
            else:  # and the other way round
                score = q[rows, h, :nope] @ w[h, :nope] @ latent.T
            score = (score + q[rows, h, nope:] @ key.T) * _scale(case)
            p = torch.softmax(torch.where(seen, score, -math.inf), 1)
            o[rows, h] = p @ (latent @ w[h, nope:].T) if decode else p @ latent @ w[h, nope:].T
    return o
