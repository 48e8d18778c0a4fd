"""The 4-bit cache in numpy and 64 bits: rotation, quantization, the page
layout and attention over it, written from the definitions in
include/drama_moe.h and independent of the kernels."""
from __future__ import annotations

import numpy as np

GROUP = 32
LIMIT = 32640.0


def bf16(x):
    """Nearest bf16 values of x, halves to even."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)


def rotate(x, positions, inv_freq, axis, interleaved):
    """x [rows, heads, D] float64, positions [axes, rows]."""
    half = len(inv_freq)
    where = positions[np.zeros(half, int) if axis is None else axis]  # [half, rows]
    angle = where.T.astype(np.float64) * inv_freq.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out = x.copy()
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def quantize(x):
    """x [..., D] -> (codes uint8 [..., D], scale words uint16 [..., D/32]), x of fp32 values."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), 0.0, np.clip(x, -LIMIT, LIMIT))
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = np.minimum(g.min(-1), 0), np.maximum(g.max(-1), 0)
    step = (hi - lo).astype(np.float32).astype(np.float64) / 15
    _, e = np.frexp(step)
    unit = np.exp2(np.maximum(e - 1, -14) - 6.0)
    s = np.ceil(step / unit) * unit
    by = np.where(s > 0, s, 1)
    z = np.minimum(np.rint(-lo / by), 15)
    c = np.clip(np.rint(g / by[..., None]) + z[..., None], 0, 15)
    words = s.astype(np.float16).view(np.uint16)
    assert not (words & 15).any() and (s.astype(np.float16) == s).all()
    return c.reshape(x.shape).astype(np.uint8), words | z.astype(np.uint16)


def value(codes, words):
    s = (words & 0xFFF0).view(np.float16).astype(np.float64)
    c = codes.reshape(*codes.shape[:-1], -1, GROUP).astype(np.float64)
    return ((c - (words & 15)[..., None]) * s[..., None]).reshape(codes.shape)


class Pages:
    """A page buffer [num_pages, kv_heads, page * (D + D/8)] of bytes."""

    def __init__(self, raw, page, dim):
        self.raw, self.page, self.dim = raw, page, dim

    def _at(self, slot):
        """Byte places, in a head's part, of a token's key codes, value codes [D/8, 4], key and value scale words."""
        p, d = self.page, self.dim
        kc = slot * (d // 2) + np.arange(d // 2)
        vc = p * d // 2 + ((slot // 4 * (d // 8) + np.arange(d // 8)) * 4 + slot % 4)[:, None] * 4 + np.arange(4)
        g = np.arange(d // GROUP)
        ks = p * d + (g * p + slot) * 2
        return kc, vc, ks, ks + p * (d // GROUP) * 2

    def put(self, page, slot, k, v):
        """k, v [kv_heads, D]."""
        kc, vc, ks, vs = self._at(slot)
        for x, codes_at, scale_at in ((k, kc, ks), (v, vc.ravel(), vs)):
            codes, words = quantize(x)
            self.raw[page][:, codes_at] = codes[:, 0::2] | codes[:, 1::2] << 4
            self.raw[page][:, scale_at] = words & 255
            self.raw[page][:, scale_at + 1] = words >> 8

    def get(self, page, slot):
        kc, vc, ks, vs = self._at(slot)
        out = []
        for codes_at, scale_at in ((kc, ks), (vc.ravel(), vs)):
            both = self.raw[page][:, codes_at]
            codes = np.stack([both & 15, both >> 4], -1).reshape(both.shape[0], self.dim)
            words = self.raw[page][:, scale_at].astype(np.uint16) | self.raw[page][:, scale_at + 1].astype(np.uint16) << 8
            out.append(value(codes, words))
        return out

    def tokens(self, table, count):
        """(k, v) [count, kv_heads, D] of a sequence's tokens; NaN on pages that are none."""
        k = np.full((count, self.raw.shape[1], self.dim), np.nan)
        v = k.copy()
        for p in range(count):
            page = table[p // self.page]
            if 0 <= page < len(self.raw):
                k[p], v[p] = self.get(page, p % self.page)
        return k, v


def attention(q, k, v, length, scale, window=0):
    """(out, weight-absolute sum, largest score uncertainty) of q [n, heads, D], the last n of `length` tokens.

    The second is sum_j p_j |v_j|, the third max_j of sum_d |q_d k_jd| * scale: what bounds of rounding errors need."""
    n, heads, dim = q.shape
    per = heads // k.shape[1]
    out, size, terms = np.zeros_like(q), np.zeros_like(q), np.zeros((n, heads))
    for i in range(n):
        place = length - n + i
        low = max(0, place - window + 1) if window else 0
        seen = np.arange(low, place + 1) if place >= 0 else np.arange(0)
        for h in range(heads):
            kk, vv = k[seen, h // per], v[seen, h // per]
            ok = ~np.isnan(kk).any(-1)
            kk, vv = kk[ok], vv[ok]
            if not len(kk):
                continue
            s = kk @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], size[i, h] = p @ vv, p @ np.abs(vv)
            terms[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return out, size, terms


def tolerance(out, size, terms, dim, tokens, eps):
    """Largest error of an attention output whose weights are rounded to fp16.

    Scores: dim products summed in fp32, each sum at most 2^-23 of the terms'
    sum off (the matrix unit may cut instead of round), and eight more
    operations of a value of that size (scale, difference from the maximum):
    delta = (dim + 8) 2^-23 terms, in a weight and in the normalising sum.
    Weights: the fp16 rounding 2^-11 (those below 2^-28 of the largest are
    subnormal and lose at most 2^-39 each) and 2^-21 of exp2.  The sums over
    the tokens, of weights and of weighted values: 2^-23 a token each.  The
    result is then rounded by at most eps / 2 of it, or, where fp16 (eps 2^-10)
    is subnormal, below 2^-14, by half of its spacing 2^-24."""
    rel = 2 * (dim + 8) * 2.0 ** -23 * terms[..., None] + 2.0 ** -11 + 2.0 ** -20 + 2 * tokens * 2.0 ** -23
    return rel * size * (1 + eps) + eps / 2 * np.abs(out) + tokens * 2.0 ** -39 * 16 + (2.0 ** -25 if eps < 2.0 ** -8 else 0.0) + 1e-30
