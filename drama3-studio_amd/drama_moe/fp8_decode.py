"""Batch-one FP8 decode entry points with the reference's signatures
(src/drama_low_vram/fp8_decode.py:114-147), on the gfx950 kernels.

``forward(kernel, x, ids, weights, staged)`` -> [1, H] in x.dtype;
``quantized_pairs(kernel, q, scales, ids, weights, staged, dtype=)`` -> ordered
fp32 partials from an activation the caller already quantized (a single
shared row, one row per pair, or one row per token of ids [T, k]; a scale for
every 128 columns, or one a row).
"""
from __future__ import annotations

import torch

from . import _lib
from .formats import FP8_DTYPE, StagedExperts, fp8_bank_struct
from .offload import DECODE_PAIRS, MAX_PAIRS, HipExpertBackend, device_state


def forward(kernel, x, ids, weights, staged: StagedExperts):
    """One input row, up to eight route slots, reference slot-order reduction."""
    return HipExpertBackend().forward(x, ids.reshape(1, -1), weights.reshape(1, -1), staged)


def quantized_pairs(kernel, q, scales, ids, weights, staged: StagedExperts, *, dtype=torch.bfloat16):
    """Ordered fp32 partials of route pairs from FP8 rows q [R, H] + scales
    [R, H/128], or [R] (also [R, 1]) for a scale a row, as
    ``norm.rms_norm(..., quant="fp8")`` gives; R == 1 shares the row across all
    pairs.  ids and weights [R, k], a prompt's routes, take each row for its k
    pairs."""
    shape, routes, hidden, device = q.shape, ids.shape, staged.hidden, staged.device
    if len(shape) != 2 or shape[1] != hidden or q.dtype not in (FP8_DTYPE, torch.uint8) or q.stride(1) != 1:
        raise ValueError(f"quantized rows must be FP8 [rows, {hidden}] with contiguous columns")
    rows = shape[0]
    routed = len(routes) == 2 and routes[0] == rows  # each row has its own k pairs
    if len(routes) != 1 or not ids.is_contiguous():
        ids = ids.reshape(-1).contiguous()
    if weights.ndim != 1 or not weights.is_contiguous():
        weights = weights.reshape(-1).contiguous()
    count = ids.shape[0]
    if count > MAX_PAIRS:
        raise ValueError(f"quantized_pairs takes at most {MAX_PAIRS} pairs per call")
    if weights.shape[0] != count:
        raise ValueError("there must be one weight per pair")
    if rows != 1 and rows != count and not routed:
        raise ValueError("quantized rows must be one shared row or one per pair, or one for each row of ids [R, k]")
    scaled = scales.shape
    groups = scaled[1] if len(scaled) == 2 else 1
    if scales.dtype is not torch.float32 or not 1 <= len(scaled) <= 2 or scaled[0] != rows or groups not in (1, hidden // 128):
        raise ValueError(f"scales must be fp32 [rows] or [rows, {hidden // 128}]")
    if q.device != device or scales.device != device or ids.device != device or weights.device != device:
        raise ValueError("rows, scales, ids, weights and experts must share a device")
    if not scales.is_contiguous():
        scales = scales.contiguous()
    out = torch.empty((count, hidden), dtype=torch.float32, device=device)
    if count == 0:
        return out
    bank = fp8_bank_struct(staged)
    state = device_state(device)
    lib = _lib.library()
    ws = state.workspace_for(lib.dmoe_fp8_workspace_bytes(bank, count))
    qb = q.view(torch.uint8)
    row_div = count if rows == 1 else routes[1] if routed else 1
    gu = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}[dtype]
    _lib.check(lib.dmoe_fp8_quantized_pairs(
        bank, _lib.ptr(qb), _lib.ptr(scales), qb.stride(0), groups, rows, row_div,
        128 if groups == hidden // 128 else hidden, _lib.ptr(ids), _lib.dtype_code(ids.dtype),
        _lib.ptr(weights), _lib.dtype_code(weights.dtype), count, gu, _lib.ptr(out), _lib.ptr(ws),
        ws.numel(), _lib.ptr(state.status), _lib.stream_handle(device)))
    return out


def staged_forward(x, ids, weights, staged: StagedExperts, *, pairs_out: bool = False,
                   gu_dtype: torch.dtype | None = None, hidden=None):
    """The decode layer as its three single-launch stages (prepare, gate/up,
    down) -- the reference's launch sequence of fp8_decode.py:114-147.

    x [T, H] float, ids / weights [T, k]; returns the slot-order combine
    [T, H] in x.dtype, or with ``pairs_out`` the ordered fp32 partials
    [T * k, H].  ``hidden`` = (hidden_q, hidden_scales) receives the FP8 hidden
    activation of stage 1 when given.
    """
    ids = ids.contiguous()
    weights = weights.contiguous()
    tokens, top_k = ids.shape
    pairs = tokens * top_k
    if pairs > DECODE_PAIRS:
        raise ValueError(f"staged_forward takes at most {DECODE_PAIRS} route pairs per call")
    if x.dim() != 2 or x.shape[0] != tokens or x.stride(1) != 1:
        raise ValueError("x must be [tokens, H] with contiguous rows")
    device = x.device
    bank = fp8_bank_struct(staged)
    inter, hsize = staged.w2_weight.shape[2], x.shape[1]
    state = device_state(device)
    lib = _lib.library()
    ws = state.workspace_for(lib.dmoe_fp8_workspace_bytes(bank, pairs))
    hq, hs = hidden if hidden is not None else (
        torch.empty(pairs, inter, dtype=torch.uint8, device=device),
        torch.empty(pairs, inter // 128, dtype=torch.float32, device=device))
    gu = _lib.dtype_code(gu_dtype or x.dtype)
    stream = _lib.stream_handle(device)
    common = (_lib.ptr(ws), ws.numel(), _lib.ptr(state.status), stream)
    _lib.check(lib.dmoe_fp8_prepare(bank, _lib.ptr(x), _lib.dtype_code(x.dtype), x.stride(0), tokens, top_k,
                                    _lib.ptr(ids), _lib.dtype_code(ids.dtype), pairs, 128, *common))
    _lib.check(lib.dmoe_fp8_gate_up(bank, top_k, pairs, 128, gu, _lib.ptr(hq), _lib.ptr(hs), *common))
    if pairs_out:
        out = torch.empty(pairs, hsize, dtype=torch.float32, device=device)
        _lib.check(lib.dmoe_fp8_down(bank, _lib.ptr(hq), _lib.ptr(hs), _lib.ptr(weights),
                                     _lib.dtype_code(weights.dtype), pairs, 1, None, _lib.F32, 0,
                                     _lib.ptr(out), *common))
    else:
        out = torch.empty(tokens, hsize, dtype=x.dtype, device=device)
        _lib.check(lib.dmoe_fp8_down(bank, _lib.ptr(hq), _lib.ptr(hs), _lib.ptr(weights),
                                     _lib.dtype_code(weights.dtype), pairs, top_k, _lib.ptr(out),
                                     _lib.dtype_code(out.dtype), out.stride(0), None, *common))
    return out
