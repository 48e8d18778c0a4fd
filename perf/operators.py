"""The attention operators over a cache held in 4 bits, as timed cases.

Three kinds of pass, each the call that a serving program makes of it:

* ``append`` -- the rows of a step or a prompt: queries and keys rotated by
  their positions (one axis, or time / height / width), keys and values
  quantized into the pages of the cache, and the values the cache then holds
  for them read back.
* ``read`` -- the keys and values of a span of a cache, as a snapshot or the
  hand-over of a prefix reads them.
* ``attend`` -- attention of new rows over the cache: one token a sequence, a
  few, a chunk behind a long past, whole prompts.

The cache: pages of ``page`` tokens; a page holds for each key/value head the
key codes [page][D/2] bytes (channel 2j in the low half of byte j), the value
codes [page/4][D/8] groups of four 32-bit words, one a token, eight channels a
word from the low bits up, then the key and the value scale words
[D/32][page] of 16 bits.  A scale word is an fp16 number of seven significant
bits, the scale s of 32 channels of a token, whose four lowest bits hold the
zero point z: a code c stands for (c - z) * s.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 32          # channels a scale
THETA = 1.0e6       # base of the rotation frequencies
# (query heads, key/value heads, head dimension)
HEADS = [(16, 2, 128), (32, 8, 128), (16, 16, 64), (16, 2, 256), (12, 4, 64), (8, 1, 128), (14, 2, 64), (8, 8, 128)]


def _attend(name, seqs, new, past, heads, *, page=64, window=0, dtype="bf16", spread=1):
    return {"name": name, "kind": "attend", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0],
            "past_hi": past[1], "hq": heads[0], "hkv": heads[1], "dim": heads[2], "page": page, "window": window,
            "dtype": dtype, "spread": spread}


def _append(name, seqs, new, past, heads, *, page=64, axes=1, rot=None, pairs=False, dtype="bf16", spread=1):
    return {"name": name, "kind": "append", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0],
            "past_hi": past[1], "hq": heads[0], "hkv": heads[1], "dim": heads[2], "page": page, "axes": axes,
            "rot": heads[2] if rot is None else rot, "pairs": pairs, "dtype": dtype, "spread": spread}


def _read(name, seqs, new, past, heads, *, page=64, dtype="bf16", spread=1):
    return {"name": name, "kind": "read", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0],
            "past_hi": past[1], "hq": heads[0], "hkv": heads[1], "dim": heads[2], "page": page, "dtype": dtype,
            "spread": spread}


def listed():
    return [
        # one stream of speech being generated, early in its text: latency alone
        _attend("decode-1-short", 1, (1, 1), (701, 701), (16, 2, 128)),
        # one stream behind a very long past
        _attend("decode-1-long", 1, (1, 1), (131070, 131070), (32, 8, 128), page=16),
        # a batched decode step of streams of all lengths
        _attend("decode-64", 64, (1, 1), (100, 8190), (32, 8, 128), page=16, spread=2),
        # small heads, each with its own keys, fp16
        _attend("decode-29-mha", 29, (1, 1), (60, 4090), (16, 16, 64), page=32, dtype="f16", spread=3),
        # proposed tokens verified, five a stream, wide heads, a sliding window
        _attend("verify-12", 12, (5, 5), (900, 12000), (16, 2, 256), window=4096, spread=4),
        # a chunk of a long prompt behind what is cached already
        _attend("chunk-2048", 1, (2048, 2048), (14336, 14336), (16, 2, 128), page=128),
        # prompts of a batch from their first token on, fp16
        _attend("prompts-9", 9, (17, 2000), (0, 0), (32, 8, 128), page=64, dtype="f16", spread=6),
        # the rows of a batched decode step
        _append("append-64", 64, (1, 1), (100, 8190), (32, 8, 128), page=16, spread=2),
        # a long prompt whose positions have three axes
        _append("append-8192", 1, (8192, 8192), (0, 0), (32, 8, 128), axes=3, spread=8),
        # prompts of odd lengths, neighbouring channels rotated, a part of the head, fp16
        _append("append-5-part", 5, (33, 901), (3, 5000), (16, 2, 256), page=32, rot=64, pairs=True, dtype="f16",
                spread=9),
        # a prefix handed to another holder
        _read("read-30001", 1, (30001, 30001), (0, 0), (32, 8, 128), page=16),
        # the last tokens of some streams
        _read("read-7", 7, (1, 300), (0, 2000), (16, 16, 64), page=32, dtype="f16", spread=12),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    heads = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    spread = rng.randrange(1000)
    kind = rng.choice(["decode", "decode", "decode", "verify", "chunk", "prompts", "append", "append", "read"])
    if kind == "decode":
        seqs = _log_int(rng, 1, 64)
        high = min(_log_int(rng, 30, 120000), 250000 // seqs)
        return _unnamed(_attend("", seqs, (1, 1), (_log_int(rng, 1, high), high), heads, page=page, dtype=dtype,
                                window=rng.choice([0, 0, 1000]), spread=spread))
    if kind == "verify":
        seqs, high = _log_int(rng, 1, 24), _log_int(rng, 30, 9000)
        return _unnamed(_attend("", seqs, (1, rng.randint(2, 9)), (_log_int(rng, 1, high), high), heads, page=page,
                                dtype=dtype, window=rng.choice([0, 0, 1000]), spread=spread))
    if kind == "chunk":
        new, past = _log_int(rng, 20, 1500), _log_int(rng, 1, 8000)
        return _unnamed(_attend("", 1, (new, new), (past, past), heads, page=page, dtype=dtype,
                                window=rng.choice([0, 0, 1000]), spread=spread))
    if kind == "prompts":
        high = _log_int(rng, 10, 1500)
        return _unnamed(_attend("", rng.randint(1, 9), (_log_int(rng, 1, high), high), (0, 0), heads, page=page,
                                dtype=dtype, spread=spread))
    if kind == "append":
        seqs, high = _log_int(rng, 1, 64), _log_int(rng, 1, 4000)
        high = min(high, 8000 // seqs)
        return _unnamed(_append("", seqs, (_log_int(rng, 1, high), high), (0, rng.choice([0, 500, 5000])), heads,
                                page=page, axes=rng.choice([1, 3]), pairs=rng.choice([True, False]),
                                rot=rng.choice([heads[2], heads[2] // 2, heads[2] // 4]), dtype=dtype, spread=spread))
    seqs, high = _log_int(rng, 1, 16), _log_int(rng, 1, 4000)
    high = min(high, 20000 // seqs)
    return _unnamed(_read("", seqs, (_log_int(rng, 1, high), high), (0, 900), heads, page=page, dtype=dtype,
                          spread=spread))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    """(new rows, past tokens) of each sequence: sizes of the case, not of a seed."""
    rng = random.Random(case["spread"] * 7919 + case["seqs"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    past = [_log_int(rng, case["past_lo"], case["past_hi"]) if case["past_lo"] else
            rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]
    return new, past


def work(case):
    new, past = _lengths(case)
    rows, hq, hkv, dim = sum(new), case["hq"], case["hkv"], case["dim"]
    token = hkv * (dim + dim // 8)  # bytes of a token in the cache: codes and scale words of its key and value
    if case["kind"] == "append":  # q in and out, k and v in, pages out, the read back
        return {"bytes": 4 * rows * hq * dim + 4 * rows * hkv * dim + 2 * rows * token + 4 * rows * hkv * dim,
                "flops": 6 * rows * (hq + hkv) * case["rot"] // 2}
    if case["kind"] == "read":
        return {"bytes": rows * token + 4 * rows * hkv * dim, "flops": 0}
    window = case["window"]
    seen = visible = 0
    for n, p in zip(new, past):
        visible += sum(min(p + i + 1, window or p + i + 1) for i in range(n))
        seen += min(p + n, window + n - 1) if window else p + n
    return {"bytes": seen * token + 4 * rows * hq * dim, "flops": 4 * dim * hq * visible}


# --------------------------------------------------------------------- inputs

def _head_bytes(case):
    return case["page"] * (case["dim"] + case["dim"] // 8)


def _random_pages(count, case, g, device):
    """Pages as a model's keys and values leave them: codes of normal values about zero points near the middle."""
    page, dim = case["page"], case["dim"]
    pool = min(count, max(1, (16 << 20) // (case["hkv"] * _head_bytes(case))))
    shape = (pool, case["hkv"])
    level = torch.special.ndtri((torch.arange(256, device=device, dtype=torch.float64) + 0.5) / 256)
    code = (level * 3.4 + 7.5).round().clamp(0, 15).to(torch.uint8)

    def half(n):
        return code[torch.randint(0, 256, (*shape, n), generator=g, device=device)]

    codes = half(page * dim) | (half(page * dim) << 4)
    scales = 0.27 * torch.exp(0.15 * torch.randn(*shape, page * dim // 16, generator=g, device=device))
    zeros = torch.randint(6, 10, scales.shape, generator=g, device=device, dtype=torch.int16)
    words = (scales.half().view(torch.int16) & -16) | zeros
    made = torch.cat([codes, words.view(torch.uint8)], -1)
    return made[torch.randint(0, pool, (count,), generator=g, device=device)]


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(int(seed))
    new, past = _lengths(case)
    seqs, rows, page, dim = case["seqs"], sum(new), case["page"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    need = [-(-(n + p) // page) for n, p in zip(new, past)]
    count = sum(need) + 3
    order = torch.randperm(count, generator=g, device=device, dtype=torch.int64).int().cpu()
    table = torch.zeros((seqs, max(need)), dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    starts = torch.zeros(seqs + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(new, dtype=torch.int32).cumsum(0)
    state = {"case": case, "pages": _random_pages(count, case, g, device), "table": table.to(device),
             "lengths": torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32).to(device),
             "starts": starts.to(device), "rows": rows, "longest": max(new), "reach": max(n + p for n, p in zip(new, past))}
    # one projection's output holds q, k and v side by side, as a fused linear leaves them
    heads = case["hq"] + 2 * case["hkv"]
    if case["kind"] != "read":
        state["qkv"] = torch.randn(rows, heads, dim, generator=g, device=device).to(dtype)
    if case["kind"] == "append":
        half = case["rot"] // 2
        state["inv_freq"] = (THETA ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(device)
        state["axis"] = (torch.arange(half) * case["axes"] // half).to(torch.uint8).to(device)
        text = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)])
        if case["axes"] == 3:  # frames of 8 by 12 patches
            shift = torch.randint(0, 50, (1,), generator=g, device=device).item()
            state["positions"] = torch.stack([text // 96 + shift, text % 96 // 12, text % 12]).to(device)
        else:
            state["positions"] = text[None].to(device)
    return state


# ------------------------------------------------------------------ plain form

def _views(pages, case):
    """(key codes, value codes, key scale words, value scale words) of the pages."""
    page, dim = case["page"], case["dim"]
    n, hkv = pages.shape[:2]
    half = page * dim // 2
    words = page * dim // 16
    return (pages[..., :half].view(n, hkv, page, dim // 2),
            pages[..., half:2 * half].view(n, hkv, page // 4, dim // 8, 4, 4),
            pages[..., 2 * half:2 * half + words].view(torch.int16).view(n, hkv, dim // GROUP, page),
            pages[..., 2 * half + words:].view(torch.int16).view(n, hkv, dim // GROUP, page))


def _values(codes, words):
    """codes [..., D/2] bytes and scale words [..., D/32] -> the 32-bit values [..., D]."""
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP))
    scale = (words & -16).view(torch.float16).float()[..., None]
    return ((both.float() - (words & 15)[..., None].float()) * scale).flatten(-2)


def _places(state):
    """(sequence, position, page, slot) of each row."""
    rows = torch.arange(state["rows"], device=state["table"].device)
    seq = torch.searchsorted(state["starts"][1:].long(), rows, right=True)
    at = state["lengths"].long()[seq] - state["starts"].long()[seq + 1] + rows
    page = state["case"]["page"]
    return seq, at, state["table"].long()[seq, at // page], at % page


def _plain_read(state):
    case = state["case"]
    kc, vc, kw, vw = _views(state["pages"], case)
    _, _, page, slot = _places(state)
    k = _values(kc[page, :, slot], kw.transpose(2, 3)[page, :, slot])
    v = _values(vc[page, :, slot // 4, :, slot % 4].flatten(2), vw.transpose(2, 3)[page, :, slot])
    return k, v


def _rotated(x, cos, sin, case):
    half = case["rot"] // 2
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    if case["pairs"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    a, b = turn[..., :half], turn[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _quantized(x):
    """x [..., D] of 32 bits -> code bytes [..., D/2], scale words [..., D/32].  Borders between codes in 64 bits."""
    x = x.double().unflatten(-1, (-1, GROUP)).clamp(-32640, 32640)
    low, high = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    step = (high - low).float().double() / 15
    unit = torch.exp2((torch.frexp(step).exponent - 1).clamp(min=-14).double() - 6)
    scale = torch.ceil(step / unit) * unit
    by = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = torch.round(-low / by).clamp(0, 15)
    code = (torch.round(x / by[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.half().view(torch.int16) | zero.to(torch.int16)


def _plain_append(state):
    case = state["case"]
    hq, hkv = case["hq"], case["hkv"]
    dtype = state["qkv"].dtype
    q, k, v = state["qkv"].split([hq, hkv, hkv], 1)
    angle = state["positions"][state["axis"].long()].T.double() * state["inv_freq"].double()
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    q_out = _rotated(q.float(), cos.float(), sin.float(), case).to(dtype)
    k = _rotated(k.double(), cos, sin, case).float()  # the key that is quantized is of 32 bits
    kc, vc, kw, vw = _views(state["pages"], case)
    _, _, page, slot = _places(state)
    codes, words = _quantized(k)
    kc[page, :, slot] = codes
    kw.transpose(2, 3)[page, :, slot] = words
    codes, words = _quantized(v.float())
    vc[page, :, slot // 4, :, slot % 4] = codes.unflatten(-1, (-1, 4))
    vw.transpose(2, 3)[page, :, slot] = words
    k, v = _plain_read(state)
    return q_out, k.half(), v.half()


def _plain_attend(state):
    case = state["case"]
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    seqs, longest, reach = case["seqs"], state["longest"], state["reach"]
    q = state["qkv"][:, :hq]
    kc, vc, kw, vw = _views(state["pages"][state["table"].long().flatten()], case)

    def whole(codes, words):  # [S * P, Hkv, page, ..] -> [S, Hkv, tokens, D]
        x = _values(codes, words.transpose(2, 3))
        return x.unflatten(0, (seqs, -1)).transpose(1, 2).flatten(2, 3)[:, :, :reach]

    keys = whole(kc, kw)
    values = whole(vc.permute(0, 1, 2, 4, 3, 5).flatten(4, 5).flatten(2, 3), vw)
    seq, at, _, _ = _places(state)
    col = torch.arange(state["rows"], device=q.device) - state["starts"].long()[seq]
    rows = q.new_zeros((seqs, longest, hq, dim), dtype=torch.float32)
    rows[seq, col] = q.float()
    where = torch.full((seqs, longest), -1, dtype=torch.int64, device=q.device)
    where[seq, col] = at
    rows = rows.transpose(1, 2).reshape(seqs, hkv, hq // hkv * longest, dim)
    score = torch.matmul(rows, keys.transpose(2, 3).contiguous()).view(seqs, hq, longest, reach) * dim ** -0.5
    token = torch.arange(reach, device=q.device)
    hidden = token > where[:, None, :, None]
    if case["window"]:
        hidden = hidden | (token <= where[:, None, :, None] - case["window"])
    score = score.masked_fill(hidden, -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(seqs, hkv, -1, reach), values).view(seqs, hq, longest, dim)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    return out.transpose(1, 2)[seq, col].to(q.dtype)


# ------------------------------------------------------------------------ runs

def _own(state):
    """The same passes through the framework's operators."""
    import os
    import sys

    place = os.path.abspath("drama3-studio_amd")
    if place not in sys.path:
        sys.path.insert(0, place)
    from drama_moe.attention import KvCache4, PagedBatch, Rotary

    case = state["case"]
    hq, hkv = case["hq"], case["hkv"]
    cache = KvCache4(state["pages"], page_size=case["page"], head_dim=case["dim"])
    batch = PagedBatch(state["table"], state["lengths"], state["starts"], rows=state["rows"],
                       max_rows=state["longest"])
    if case["kind"] == "read":
        return cache.read(batch, dtype=torch.float16)
    qkv = state["qkv"]
    if case["kind"] == "attend":
        return cache.attend(qkv[:, :hq], batch, window=case["window"])
    rotary = Rotary(state["inv_freq"], axis=state["axis"], interleaved=case["pairs"])
    q = cache.append(qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], batch, q=qkv[:, :hq], rotary=rotary,
                     positions=state["positions"])
    return (q, *cache.read(batch, dtype=torch.float16))


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "append":
        return _plain_append(state)
    if kind == "read":
        k, v = _plain_read(state)
        return k.half(), v.half()
    return _plain_attend(state)


# ----------------------------------------------------------------------- exact

def _token_values(state, pick):
    """64-bit (k, v) [n, Hkv, D] of the (sequence, position) pairs, from the layout's definition, channel by channel."""
    case = state["case"]
    page, dim = case["page"], case["dim"]
    seq, at = pick
    raw = state["pages"]
    where = state["table"].long()[seq, at // page]
    slot = (at % page)[:, None, None]
    channel = torch.arange(dim, device=raw.device)
    heads = torch.arange(case["hkv"], device=raw.device)[None, :, None]
    where = where[:, None, None]
    half, words = page * dim // 2, page * dim // 16

    def byte(offset):
        return raw[where, heads, offset].int()

    def value(code_at, scale_base):
        code = (byte(code_at) >> (4 * (channel % 2))) & 15
        base = scale_base + 2 * (channel // GROUP * page + slot)
        word = byte(base) | (byte(base + 1) << 8)
        exponent, mantissa = (word >> 10) & 31, word & 1008
        scale = torch.where(exponent > 0, (1024 + mantissa).double() * torch.exp2(exponent.double() - 25),
                            mantissa.double() * 2.0 ** -24)
        return (code - (word & 15)).double() * scale

    k = value(slot * (dim // 2) + channel // 2, 2 * half)
    v = value(half + ((slot // 4 * (dim // 8) + channel // 8) * 4 + slot % 4) * 4 + channel % 8 // 2, 2 * half + words)
    return k, v


def _nearest(x):
    """The values of the codes nearest to x [..., D], by the definition."""
    x = x.clamp(-32640, 32640).unflatten(-1, (-1, GROUP))
    low = torch.minimum(x.min(-1, keepdim=True).values, x.new_zeros(()))
    high = torch.maximum(x.max(-1, keepdim=True).values, x.new_zeros(()))
    step = ((high - low).float().double() / 15).clamp(min=2.0 ** -40)
    digits = torch.exp2(torch.floor(torch.log2(step)).clamp(min=-14) - 6)
    scale = torch.ceil(step / digits) * digits
    zero = torch.round(-low / scale).clamp(0, 15)
    value = (torch.round(x / scale) + zero).clamp(0, 15) - zero
    return torch.where(high > low, value * scale, torch.zeros_like(value)).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    new, past = _lengths(case)
    device = state["pages"].device
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if case["kind"] == "attend":
        out, at = [], 0
        for b, (n, p) in enumerate(zip(new, past)):
            tokens = torch.arange(n + p, device=device)
            parts = [_token_values(state, (torch.full_like(t, b), t)) for t in tokens.split(8192)]
            k, v = (torch.cat([x[i] for x in parts]) for i in (0, 1))
            q = state["qkv"][at:at + n, :hq].double()
            at += n
            mine = torch.empty(n, hq, dim, dtype=torch.float64, device=device)
            for h in range(hq):
                s = q[:, h] @ k[:, h * hkv // hq].T * dim ** -0.5
                row = (p + torch.arange(n, device=device))[:, None]
                seen = tokens <= row
                if case["window"]:
                    seen &= tokens > row - case["window"]
                mine[:, h] = torch.softmax(s.where(seen, torch.full_like(s, -math.inf)), -1) @ v[:, h * hkv // hq]
            out.append(mine)
        return torch.cat(out)
    if case["kind"] == "read":
        seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)]).to(device)
        at = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)]).to(device)
        parts = [_token_values(state, (s, a)) for s, a in zip(seq.split(8192), at.split(8192))]
        return tuple(torch.cat([x[i] for x in parts]) for i in (0, 1))
    q, k, v = (x.double() for x in state["qkv"].split([hq, hkv, hkv], 1))
    half = case["rot"] // 2
    turn = torch.arange(half, device=device)
    first, second = (2 * turn, 2 * turn + 1) if case["pairs"] else (turn, turn + half)
    phase = torch.polar(torch.ones((), dtype=torch.float64, device=device), state["positions"].double().T[:, state["axis"].long()] *
                        state["inv_freq"].double())[:, None]

    def rotate(x):
        z = torch.complex(x[..., first], x[..., second]) * phase
        x = x.clone()
        x[..., first], x[..., second] = z.real, z.imag
        return x

    return rotate(q), _nearest(rotate(k).float().double()), _nearest(v)
