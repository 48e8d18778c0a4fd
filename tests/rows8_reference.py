"""Rows and products in 8 bits in numpy and 64 bits, written from the
definitions in include/drama_moe.h and independent of the kernels."""
from __future__ import annotations

import numpy as np
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
SMALL = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the smallest step


def wide(t):
    return t.detach().cpu().double().numpy()


def through(x, dtype):
    """x float64 rounded once to ``dtype`` (by way of an odd fp32, so that nothing is rounded twice)."""
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        f = x.astype(np.float32)
    if dtype is torch.float32:
        return f.astype(np.float64)
    bits = f.view(np.uint32).copy()
    off = np.isfinite(f) & (f.astype(np.float64) != x)
    bits -= (off & (np.abs(f.astype(np.float64)) > np.abs(x))).astype(np.uint32)
    bits |= off.astype(np.uint32)
    return torch.from_numpy(bits.view(np.float32).copy()).to(dtype).double().numpy()


def norm(x, residual, weight, dtype, *, eps, offset=0.0):
    """(h, y) float64 of float64 rows that hold values of ``dtype``."""
    h = x if residual is None else through(x + residual, dtype)
    gain = (np.float32(offset) + weight.astype(np.float32)).astype(np.float32).astype(np.float64)
    u = (h * gain).astype(np.float32).astype(np.float64)
    return h, u * (1.0 / np.sqrt((h * h).mean(-1, keepdims=True) + eps))


def int8(y):
    """(codes, scales) float64 of rows y float64; rows that are not finite give 0 and NaN."""
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.abs(y).max(-1).astype(np.float32)
    fine = np.isfinite(top)
    scale = np.maximum(np.where(fine, top, 0), np.float32(1e-12)) * (np.float32(1) / np.float32(127))
    with np.errstate(invalid="ignore"):
        codes = np.clip(np.rint(y / scale.astype(np.float64)[:, None]), -127, 127)
    codes[~fine] = 0
    scale = scale.astype(np.float64)
    scale[~fine] = np.nan
    return codes, scale


E4M3 = np.array([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def e4m3(y, group):
    """(numbers, scales) of groups of columns, ties to the even code."""
    rows = y.shape[0]
    y = y.reshape(rows, -1, group)
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.abs(y).max(-1).astype(np.float32)
    fine = np.isfinite(top)
    scale = (np.maximum(np.where(fine, top, 0), np.float32(1e-10)) * np.float32(1 / 448)).astype(np.float32)
    with np.errstate(invalid="ignore"):
        size = np.abs(y / scale.astype(np.float64)[..., None])
    size[~fine] = 0
    middle = (E4M3[1:] + E4M3[:-1]) / 2
    low, high = np.searchsorted(middle, size, "left"), np.searchsorted(middle, size, "right")
    at = np.where((low != high) & (low % 2 == 1), high, low)
    values = np.where(fine[..., None], np.copysign(E4M3[at], y), 0)
    scale = scale.astype(np.float64)
    scale[~fine] = np.nan
    return values.reshape(rows, -1), scale


def product(codes, scales, w, w_scales, bias=None, residual=None):
    """(result, magnitude that its fp32 steps are relative to), float64."""
    p = (codes @ w.T) * w_scales * scales[:, None]
    out, size = p.copy(), np.abs(p)
    for more in (bias, residual):
        if more is not None:
            out = out + more
            size = size + np.abs(more)
    return out, size


def act(z, name):
    y = z if name == "silu" else 2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)
    with np.errstate(over="ignore"):
        return z / (1 + np.exp(-y)), y


def feed_forward(codes, scales, w, w_scales, down, down_scales, dtype, name, residual=None):
    """(low, high) float64: where each output lies before its own rounding.

    The fp32 steps of the hidden rows are off by less than ``unsure``, which
    may move a value across a border of ``dtype`` or of two codes, and the
    largest of a row its scale; everything that this can lead to is between
    the bounds."""
    first, _ = product(codes, scales, w, w_scales)
    inter = first.shape[1] // 2
    gate, up = first[:, :inter], first[:, inter:]
    value, y = act(gate, name)
    hidden = value * up
    # three products of two roundings, the polynomial's and the exponential's relative error (which grows with its
    # argument) and the quotient's
    unsure = 2.0 ** -20 + (np.abs(y) + 1) * 2.0 ** -21
    size = np.abs(hidden)
    low, high = through(size * (1 - unsure), dtype), through(size * (1 + unsure), dtype)
    s_low, s_high = int8(low)[1][:, None], int8(high)[1][:, None]
    c_low, c_high = np.clip(np.rint(low / s_high), 0, 127), np.clip(np.rint(high / s_low), 0, 127)
    # |code * scale| lies in [a, b]
    a, b = c_low * s_low, c_high * s_high
    sign = np.sign(hidden)
    lo, hi = np.where(sign >= 0, a, -b), np.where(sign >= 0, b, -a)
    up_w, down_w = np.maximum(down, 0), np.minimum(down, 0)
    first_lo, first_hi = lo @ up_w.T + hi @ down_w.T, hi @ up_w.T + lo @ down_w.T
    first_lo, first_hi = first_lo * down_scales, first_hi * down_scales
    size = np.maximum(np.abs(first_lo), np.abs(first_hi))
    if residual is not None:
        first_lo, first_hi, size = first_lo + residual, first_hi + residual, size + np.abs(residual)
    slack = 6 * 2.0 ** -24 * size
    return first_lo - slack, first_hi + slack
