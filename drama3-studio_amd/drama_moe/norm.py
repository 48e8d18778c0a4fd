"""Root-mean-square norm with the residual's addition, and the next block's
input in 8 bits.

What stands between two blocks of a decoder layer: the block's output is
added to the residual stream, the sum is normalised, and what the next block
reads leaves in its own form -- rows as they are (a router, ``MoeBlock``), 8-bit
integers with a scale a row (``int8.Int8Linear``, ``int8.Int8FeedForward``), or
E4M3 with a scale a row or for every 128 columns
(``fp8_decode.quantized_pairs``, for single rows and prompts) -- in one pass over the rows.  In the
reference these are torch modules of the model it drives
(src/drama_low_vram/backbone_graph.py:297-316).  Serving only: with gradients
enabled, inputs that need them are refused, and inputs with a forward-mode
tangent always.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import _lib
from .attention import _on, _stream
from .int8 import (_FLOATS, E4M3, E4M3_GROUP, GROUP, INT8, QuantRows, _check_float, _check_sizes, _desc, _flat, _gpu,
                   _no_gradients, _same_device, _status)

QUANT_FORMATS = {"int8": INT8, "fp8": E4M3, "fp8-128": E4M3_GROUP}


class Normed(NamedTuple):
    """``hidden``: x + residual (x itself without one); ``rows``: the normalised
    rows or None; ``quant``: them in 8 bits or None."""

    hidden: Tensor
    rows: Tensor | None
    quant: QuantRows | None


def rms_norm(x: Tensor, weight: Tensor, *, residual: Tensor | None = None, eps: float = 1e-6, offset: float = 0.0,
             quant: str | None = None, rows: bool | None = None) -> Normed:
    """h = x + residual, rounded to their type; y = h (offset + weight) / sqrt(mean(h^2) + eps).

    x [..., columns] and residual have one type (bf16, fp16, fp32), weight
    [columns] any of them.  ``quant`` asks for y in 8 bits ("int8", "fp8",
    "fp8-128"), as rows of all leading dimensions; ``rows`` for y itself
    (default: without ``quant``).  Sums and roots are of 64 bits, products of 32,
    and the codes are of y before its rounding to the rows' type.  A row with an infinity or NaN gets codes
    of 0 and a scale of NaN, and raises the device status bit."""
    fmt = None
    if quant is not None:
        fmt = QUANT_FORMATS.get(quant)
        if fmt is None:
            raise ValueError(f"quant must be one of {sorted(QUANT_FORMATS)}")
    if rows is None:
        rows = fmt is None
    elif not rows and fmt is None:
        raise ValueError("the norm has no output: neither rows nor quant")
    _no_gradients("x weight residual", x, weight, residual)
    flat = _flat(x, "x")
    count, cols = flat.shape
    _check_sizes(count, cols)
    if weight.shape != (cols,):
        raise ValueError(f"weight must be [{cols}]")
    dtype, shape = x.dtype, x.shape
    if weight.dtype not in _FLOATS:
        _check_float(weight, "weight")
    if fmt == E4M3_GROUP and cols % GROUP:
        raise ValueError("groups of 128 need a multiple of 128 columns")
    add = None
    if residual is not None:
        if residual.shape != shape or residual.dtype is not dtype:
            raise ValueError(f"residual must be {dtype} {list(shape)}")
        add = _flat(residual, "residual")
    device = _gpu(x.device, x)
    _same_device(device, weight=weight, residual=residual)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    hidden = x if add is None else flat.new_empty((count, cols))
    y = flat.new_empty((count, cols)) if rows else None
    q = QuantRows._new(count, cols, fmt, device) if fmt is not None else None
    if count:
        code = _FLOATS[dtype]
        with _on(device):
            _lib.check(_lib.library().dmoe_rms_norm(
                _desc(flat), _desc(add) if add is not None else None, count, cols, weight.data_ptr(),
                _FLOATS[weight.dtype], offset, eps, _lib.Rows(hidden.data_ptr(), cols, code) if add is not None else None,
                _lib.Rows(y.data_ptr(), cols, code) if rows else None, q.desc if q is not None else None,
                _status(device), _stream(device)))
    if len(shape) != 2:
        if add is not None:
            hidden = hidden.view(shape)
        if rows:
            y = y.view(shape)
    return Normed(hidden, y, q)


class RmsNorm(torch.nn.Module):
    """``rms_norm`` with a weight of its own (a constant); ``quant`` and
    ``rows`` are those of ``rms_norm``."""

    def __init__(self, weight: Tensor, *, eps: float = 1e-6, offset: float = 0.0, quant: str | None = None,
                 rows: bool | None = None):
        super().__init__()
        if weight.ndim != 1:
            raise ValueError("weight must be [columns]")
        if quant is not None and quant not in QUANT_FORMATS:
            raise ValueError(f"quant must be one of {sorted(QUANT_FORMATS)}")
        self.register_buffer("weight", weight.detach())
        self.eps, self.offset, self.quant, self.rows = float(eps), float(offset), quant, rows

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Normed:
        return rms_norm(x, self.weight, residual=residual, eps=self.eps, offset=self.offset, quant=self.quant, rows=self.rows)
