"""A paged key/value cache in 4 bits, attention over it, and keys rotated on
their way into a cache, as cases that can be timed and checked.

The 4-bit cache holds, per token and KV head, keys and values in groups of 64
elements (the last one may be shorter) with a bf16 scale s and a bf16 offset m,

  s = max((max - min) / 15, FLT_MIN),  m = min + 8 s,
  code = round half to even(clamp((x - m) / s, -8, 7)),  x ~ s code + m;

the 8-bit one a row of int8 with one fp32 scale, s = max(absmax / 127, FLT_MIN),
code = round half away(clamp(x / s, -127, 127)).  Attention is causal:

  o[i, h] = sum_t softmax_t(q[i, h] . k_t / sqrt(d))[t] v_t * sigmoid(gate[i, h]).

Three kinds, each one pass through the public entry points of qm38.Runtime:

  append   rows of several sequences behind what they cache, in 4 or 8 bits,
           keys and queries rotated on the way; then the new rows read back
                                              kv_append, KvCache.load
  decode   one new token for each sequence of a ragged batch over 4-bit caches
           rotate: from a fused projection    kv_append, gqa_attention
           else: from prepared rows           gqa_attention_q8
  prefill  new rows of one sequence over its 4-bit cache
           rotate: from a fused projection    kv_append, gqa_attention_prefill
           else: from prepared rows           gqa_attention_q8_prefill

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
FLT_MIN = 1.1754943508222875e-38
THETA = 1e6
GROUP = 64

# (query heads, KV heads, head dim): the benchmark's attention layer, the gated
# layer of a hybrid model, narrow heads, and heads that fill no tile.
LAYER, GATED, NARROW, ODD = (64, 8, 128), (24, 4, 256), (32, 8, 64), (20, 5, 80)


def _shape(shape):
    return dict(zip(("heads", "kv_heads", "dim"), shape))


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # The step of one decoding request into its cache: latency.
        dict(name="append_1", kind="append", bits=4, rows="1", cached="1000", layout="half", scaling="none", **_shape(LAYER)),
        # A scheduler's step: drafts, single tokens, prompts and an idle request.
        dict(name="append_ragged_q8", kind="append", bits=8, rows="333,1,5,0,700,17", cached="0,4095,20001,64,16,999",
             layout="half", scaling="yarn", **_shape(GATED)),
        # A long prompt's chunk.
        dict(name="append_8192", kind="append", bits=4, rows="8192", cached="4001", layout="interleaved", scaling="linear",
             **_shape(LAYER)),
        # One young request of a hybrid model: latency.
        dict(name="decode_500", kind="decode", rotate=False, gated=True, cached="500", **_shape(GATED)),
        # One request at the benchmark's context.
        dict(name="decode_32k", kind="decode", rotate=False, gated=False, cached="32768", **_shape(LAYER)),
        # A long document, no page full.
        dict(name="decode_128k", kind="decode", rotate=True, gated=True, cached="131071", **_shape(GATED)),
        # Requests of very different ages in one batch, one of them new.
        dict(name="decode_ragged", kind="decode", rotate=False, gated=False,
             cached="4096,32768,131072,777,65535,16000,0,8191", **_shape(LAYER)),
        # A served batch of a model with narrow heads.
        dict(name="decode_served", kind="decode", rotate=True, gated=False,
             cached=",".join(str(200 + 137 * i) for i in range(24)), **_shape(NARROW)),
        # Verification of a few drafted tokens at a long context.
        dict(name="prefill_5_on_20001", kind="prefill", rotate=False, gated=True, rows=5, cached="20001", **_shape(GATED)),
        # A short prompt, no size a multiple of a tile's.
        dict(name="prefill_333", kind="prefill", rotate=True, gated=False, rows=333, cached="0", **_shape(ODD)),
        # A prompt's first chunk.
        dict(name="prefill_1000", kind="prefill", rotate=True, gated=True, rows=1000, cached="0", **_shape(GATED)),
        # A prompt's second chunk.
        dict(name="prefill_2048_on_4096", kind="prefill", rotate=True, gated=False, rows=2048, cached="4096", **_shape(LAYER)),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    shape = _shape(rng.choice([LAYER, LAYER, GATED, GATED, NARROW, ODD]))
    if kind == "append":
        n = rng.randint(1, 6)
        return dict(kind=kind, bits=rng.choice([4, 4, 8]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "yarn"]),
                    rows=",".join(str(_log_int(rng, 1, 8192 // n)) for _ in range(n)),
                    cached=",".join(str(_log_int(rng, 1, 20000) - 1) for _ in range(n)), **shape)
    rest = dict(kind=kind, rotate=rng.random() < 0.5, gated=rng.random() < 0.5, **shape)
    if kind == "decode":
        # No more tokens than the listed ragged batch's.
        lengths = [_log_int(rng, 1, 65536) - 1 for _ in range(rng.randint(1, 9))]
        while sum(lengths) > 250000:
            lengths.remove(max(lengths))
        return dict(cached=",".join(map(str, lengths)), **rest)
    rows = _log_int(rng, 2, 2048)
    # No more than the listed long prompt's products.
    cached = min(_log_int(rng, 1, 32768) - 1, int(8e10 / (rows * shape["heads"] * shape["dim"])) - rows // 2)
    return dict(rows=rows, cached=str(max(0, cached)), **rest)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _rows(case):
    """New rows of every sequence."""
    if case["kind"] == "append":
        return _numbers(case["rows"])
    return [1] * len(_numbers(case["cached"])) if case["kind"] == "decode" else [case["rows"]]


# ---------------------------------------------------------------------------
# Inputs, made from the seed alone
# ---------------------------------------------------------------------------
def _inputs(case, seed):
    """What both sides and exact() start from."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    rows, cached = _rows(case), _numbers(case["cached"])
    total = sum(rows)
    s = dict(case=case, rows=rows, cached=cached)
    # Keys have means of their own in every channel, which rotation mixes pairwise.
    mean = randn(KVH, D)
    # The cached tokens' rows, rotated already.
    s["old"] = [((randn(n, KVH, D) + mean).to(torch.bfloat16), randn(n, KVH, D).to(torch.bfloat16)) for n in cached]
    q, k, v = 1.5 * randn(total, H, D), randn(total, KVH, D) + mean, randn(total, KVH, D)
    if case["kind"] == "append" or case["rotate"]:
        # Rows of a fused projection: queries, keys, values.
        s["qkv"] = torch.cat([x.flatten(1) for x in (q, k, v)], 1).to(torch.bfloat16)
    else:
        s["q"], s["k"], s["v"] = q.to(torch.bfloat16), k, v
    if case["kind"] == "append":
        s["positions"] = torch.randint(0, 131072, (total,), generator=gen, device=DEV, dtype=torch.int32)
    elif case["gated"]:
        s["gate"] = randn(total, H, D).to(torch.bfloat16)
    return s


def _rotary_dim(case):
    # Half of the hybrid model's head turns, all of the others'.
    return case["dim"] // 2 if case["dim"] == 256 else case["dim"]


def _scaling(case):
    return case.get("scaling", "none")


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
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    bits = case.get("bits", 4)
    if own:
        qm38, rt = _library()
        s["rt"] = rt
        s["rotary"] = qm38.RotaryConfig(
            rotary_dim=_rotary_dim(case), interleaved=case.get("layout") == "interleaved", theta=THETA,
            scaling=_scaling(case), factor=4.0, original_positions=16384)
        s["caches"] = []
        for (k, v), new in zip(s["old"], s["rows"]):
            cache = rt.create_q4_kv_state(KVH, D) if bits == 4 else rt.create_q8_kv_state(KVH, D)
            cache.reserve(len(k) + new)
            if len(k):
                rt.kv_append([cache], [len(k)], k, v)
            s["caches"].append(cache)
        total = sum(s["rows"])
        if "qkv" in s:
            s["q_out"] = torch.empty(total, H, D, dtype=torch.bfloat16, device=DEV)
        if case["kind"] == "append":
            s["read"] = [[torch.empty(n, KVH, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)] for n in s["rows"]]
        else:
            s["o"] = torch.empty(total, H, D, dtype=torch.bfloat16, device=DEV)
        return s
    # One padded cache for the batch, with room for the new rows.
    room = max(n + new for n, new in zip(s["cached"], s["rows"]))
    s["cache"] = []
    for part in (0, 1):
        codes = torch.zeros(len(s["cached"]), room, KVH, D, dtype=torch.int8, device=DEV)
        groups = -(-D // GROUP) if bits == 4 else 1
        scale, offset = (torch.zeros(len(s["cached"]), room, KVH, groups, device=DEV) for _ in range(2))
        for b, old in enumerate(s["old"]):
            n = len(old[part])
            codes[b, :n], scale[b, :n], offset[b, :n] = _quantised(old[part].float(), bits)
        s["cache"].append((codes, scale, offset))
    s["length"] = torch.tensor(s["cached"], device=DEV)
    # Where each new row goes, and what position it has.
    s["seq"] = torch.cat([torch.full((n,), b, device=DEV) for b, n in enumerate(s["rows"])])
    s["token"] = torch.cat([torch.arange(n, device=DEV) + at for at, n in zip(s["cached"], s["rows"])])
    return s


# ---------------------------------------------------------------------------
# The plain forms, in 32 bits (angles and the rotation of keys, whose codes may
# lie on a border, in 64)
# ---------------------------------------------------------------------------
def _frequencies(case):
    """Turns per position of every frequency, and the factor of sine and cosine, in 64 bits."""
    rd = _rotary_dim(case)
    i = torch.arange(rd // 2, dtype=torch.float64, device=DEV)
    freq = THETA ** (-2 * i / rd)
    if _scaling(case) == "linear":
        return freq / 4.0, 1.0
    if _scaling(case) == "yarn":
        # Frequencies that turn often within the original context stay, slow
        # ones are divided by the factor, a ramp between them.
        low, high = (rd * math.log(16384 / (turns * 2 * math.pi)) / (2 * math.log(THETA)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rd - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        # (the library takes the factor of sine and cosine in 32 bits)
        return freq / 4.0 * ramp + freq * (1 - ramp), torch.tensor(0.1 * math.log(4.0) + 1.0).item()
    return freq, 1.0


def _turned(x, positions, case):
    """x [rows][heads][dim] in 64 bits, its first elements rotated."""
    rd = _rotary_dim(case)
    freq, factor = _frequencies(case)
    angle = positions.double()[:, None, None] * freq
    cos, sin = torch.cos(angle) * factor, torch.sin(angle) * factor
    part, rest = x[..., :rd].double(), x[..., rd:].double()
    if case.get("layout") == "interleaved":
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :rd // 2], part[..., rd // 2:]
        part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((part, rest), -1)


def _over(x, number):
    # (by a Python number torch multiplies with its reciprocal)
    return x / torch.full_like(x, number)


def _quantised(x, bits):
    """Codes, scales and offsets of fp32 rows [...][dim], one scale a group."""
    if bits == 8:
        scale = _over(x.abs().amax(-1, keepdim=True), 127).clamp(min=FLT_MIN)
        t = (x / scale).clamp(-127, 127).double()  # adding a half in 32 bits would round up what is just below it
        return (torch.sign(t) * torch.floor(t.abs() + 0.5)).to(torch.int8), scale, torch.zeros_like(scale)
    codes, scales, offsets = [], [], []
    for part in x.split(GROUP, -1):
        low, high = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
        scale = _over(high * 0.5 - low * 0.5, 7.5).clamp(min=FLT_MIN).to(torch.bfloat16).float()
        offset = (low + scale * 8).to(torch.bfloat16).float()
        codes.append(torch.round(((part - offset) / scale).clamp(-8, 7)).to(torch.int8))
        scales.append(scale)
        offsets.append(offset)
    return torch.cat(codes, -1), torch.cat(scales, -1), torch.cat(offsets, -1)


def _held(codes, scale, offset):
    """What codes stand for, in fp32."""
    if scale.shape[-1] == 1:
        return codes.float() * scale + offset
    per = [codes[..., GROUP * g:GROUP * (g + 1)].float() * scale[..., g:g + 1] + offset[..., g:g + 1]
           for g in range(scale.shape[-1])]
    return torch.cat(per, -1)


def _plain_append(s):
    """The new rows' codes behind every sequence's cached ones; returns the rotated queries."""
    case = s["case"]
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    if "qkv" in s:
        q, k, v = (x.unflatten(1, (-1, D)) for x in s["qkv"].split([H * D, KVH * D, KVH * D], 1))
        positions = s.get("positions", s["token"])
        q, k, v = _turned(q, positions, case).to(torch.bfloat16), _turned(k, positions, case).float(), v.float()
    else:
        q, k, v = s["q"], s["k"], s["v"]
    for x, cache in zip((k, v), s["cache"]):
        for held, new in zip(cache, _quantised(x, case.get("bits", 4))):
            held[s["seq"], s["token"]] = new
    return q


def _plain_load(s):
    out = []
    for b, (at, n) in enumerate(zip(s["cached"], s["rows"])):
        out.append([_held(*(x[b, at:at + n] for x in cache)).to(torch.bfloat16) for cache in s["cache"]])
    return out


def _softmax(x):
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_attention(s, q):
    """Every row over its sequence's tokens up to its own."""
    case = s["case"]
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    k, v = (_held(*cache).transpose(1, 2).contiguous() for cache in s["cache"])  # [B][KVH][T][D]
    B = len(s["cached"])
    # [B][KVH][rows and heads of the group][D]
    rows = q.float().unflatten(0, (B, -1)).unflatten(2, (KVH, -1)).transpose(1, 2)
    shape = rows.shape
    score = torch.matmul(rows.flatten(2, 3), k.transpose(2, 3).contiguous()) / math.sqrt(D)
    hidden = torch.arange(k.shape[2], device=DEV) > s["token"].view(B, -1, 1)  # [B][rows][T]
    score = score.unflatten(2, shape[2:4]).masked_fill(hidden[:, None, :, None], -math.inf).flatten(2, 3)
    o = torch.matmul(_softmax(score), v).view(shape).transpose(1, 2).reshape(q.shape)
    if "gate" in s:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return o.to(torch.bfloat16)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind, H, KVH, D = (case[key] for key in ("kind", "heads", "kv_heads", "dim"))
    if not own:
        q = _plain_append(s)
        return (q, _plain_load(s)) if kind == "append" else _plain_attention(s, q)
    rt, caches, gate = s["rt"], s["caches"], s.get("gate")
    for cache, length in zip(caches, s["cached"]):
        cache.truncate(length)
    if "qkv" in s:
        q, k, v = s["qkv"].split([H * D, KVH * D, KVH * D], 1)
        rt.kv_append(caches, s["rows"], k, v, rotary=s["rotary"], positions=s.get("positions"),
                     q=q, q_out=s["q_out"], num_heads=H)
    if kind == "append":
        for cache, length, n, (k, v) in zip(caches, s["cached"], s["rows"], s["read"]):
            if n:
                cache.load(length, n, k, v)
        return s["q_out"], s["read"]
    if kind == "decode":
        if case["rotate"]:
            rt.gqa_attention(caches, s["q_out"], gate, H, s["o"])
        else:
            rt.gqa_attention_q8(caches, s["q"], gate, s["k"], s["v"], H, s["o"])
    elif case["rotate"]:
        rt.gqa_attention_prefill(caches[0], s["q_out"], gate, H, case["rows"], s["o"])
    else:
        rt.gqa_attention_q8_prefill(caches[0], s["q"], gate, s["k"], s["v"], H, case["rows"], s["o"])
    return s["o"]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    rows, cached = _rows(case), _numbers(case["cached"])
    total = sum(rows)
    # Bytes of a token in the cache, and of a row's queries, keys and values as given.
    held = 2 * KVH * (D / 2 + 4 * -(-D // GROUP) if case.get("bits", 4) == 4 else D + 4)
    fused = case["kind"] == "append" or case["rotate"]
    given = 2 * H * D + (4 if fused else 8) * KVH * D
    turned = 3 * total * (H + KVH) * _rotary_dim(case) if fused else 0
    if case["kind"] == "append":
        # Rows in, queries and codes out; codes in, keys and values out.
        return {"bytes": total * (given + 4 + 2 * H * D + 2 * held + 4 * KVH * D), "flops": turned + 12 * total * KVH * D}
    seen = sum(n * at + n * (n + 1) // 2 for n, at in zip(rows, cached))  # (row, visible token) pairs
    return {"bytes": sum(cached) * held + total * (given + held + (4 if case["gated"] else 2) * H * D),
            "flops": 4 * seen * H * D + turned}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_turned(x, positions, case):
    rd = _rotary_dim(case)
    freq, factor = _frequencies(case)
    turn = torch.polar(torch.full_like(freq, factor).expand(len(x), -1), positions.double()[:, None] * freq)[:, None]
    x = x.double()
    if not len(x):
        return x
    part = x[..., :rd]
    interleaved = case.get("layout") == "interleaved"
    pair = part.unflatten(-1, (-1, 2)) if interleaved else part.unflatten(-1, (2, -1)).transpose(-1, -2)
    pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    return torch.cat(((pair if interleaved else pair.transpose(-1, -2)).flatten(-2), x[..., rd:]), -1)


def _exact_held(x, bits):
    """What the cache stands for after these rows [n][KVH][D]."""
    x = x.double()
    if bits == 8:
        step = torch.clamp(x.abs().max(-1, keepdim=True).values / 127.0, min=FLT_MIN)
        t = x / step
        return torch.where(t < 0, torch.ceil(t - 0.5), torch.floor(t + 0.5)) * step
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], GROUP):
        part = x[..., at:at + GROUP]
        least, most = torch.aminmax(part, dim=-1, keepdim=True)
        step = torch.clamp((most - least) / 15.0, min=FLT_MIN).to(torch.bfloat16).double()
        middle = (least + 8.0 * step).to(torch.bfloat16).double()
        out[..., at:at + GROUP] = torch.clamp(torch.round((part - middle) / step), -8, 7) * step + middle
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    bits, first, out, turned = case.get("bits", 4), 0, [], []
    for b, (at, n) in enumerate(zip(s["cached"], s["rows"])):
        mine = slice(first, first + n)
        first += n
        if "qkv" in s:
            x = s["qkv"][mine].unflatten(1, (H + 2 * KVH, D))
            positions = s["positions"][mine] if "positions" in s else torch.arange(at, at + n, device=DEV)
            q, k, v = _exact_turned(x[:, :H], positions, case), _exact_turned(x[:, H:H + KVH], positions, case), x[:, H + KVH:]
        else:
            q, k, v = s["q"][mine].double(), s["k"][mine], s["v"][mine]
        if case["kind"] == "append":
            turned.append(q)
            out.append([_exact_held(k, bits), _exact_held(v, bits)])
            continue
        if "qkv" in s:
            q = q.to(torch.bfloat16).double()  # as attention is given them
        o = torch.empty(n, H, D, dtype=torch.float64, device=DEV)
        seen = torch.ones(n, at + n, dtype=torch.bool, device=DEV).tril(at)
        for g in range(KVH):
            keys = torch.cat((_exact_held(s["old"][b][0][:, g], bits), _exact_held(k[:, g], bits)))
            values = torch.cat((_exact_held(s["old"][b][1][:, g], bits), _exact_held(v[:, g], bits)))
            for h in range(g * (H // KVH), (g + 1) * (H // KVH)):
                score = torch.where(seen, q[:, h] @ keys.T * D ** -0.5, -math.inf)
                o[:, h] = torch.softmax(score, 1) @ values
        if "gate" in s:
            o = o * torch.sigmoid(s["gate"][mine].double())
        out.append(o)
    return (torch.cat(turned), out) if case["kind"] == "append" else torch.cat(out)
