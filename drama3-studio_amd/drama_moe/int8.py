"""Rows and matrices of 8-bit integers: the dense linears and feed-forward
blocks of a decoder layer beside its routed experts.

``QuantRows`` are rows in 8 bits with their scales, as ``quantize_rows`` and
``norm.rms_norm`` make them: integers or E4M3 with a scale a row, or E4M3
with a scale for every 128 columns (``fp8_decode.quantized_pairs`` takes
E4M3 rows of both kinds).  ``Int8Weight`` is a matrix of 8-bit integers with a scale for each
output channel.  ``int8_linear`` multiplies the two, ``int8_feed_forward``
runs a gated feed-forward block on two such matrices; ``Int8Linear`` and
``Int8FeedForward`` are the modules, ``Int8Linear`` next to
``quantized.GPTQLinear``.  Sums are exact in 32-bit integers; scales, bias,
residual and activation are applied in fp32 and rounded once.

The reference keeps its dense linears in bf16 or GPTQ
(src/drama_low_vram/quantized_model.py:71-91).  No call synchronizes the host,
every call can be captured in a hipGraph, and scratch is allocated for each
call by torch.  Matrices are constants: there is no backward, and with
gradients enabled inputs that need them are refused, and inputs with a
forward-mode tangent always.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _lib
from .attention import _LEVEL, _on, _refusal, _stream
from .formats import FP8_DTYPE, HeldTypes
from .offload import _STATES, _device_of, device_state

MAX_K = 65536
MAX_ROWS = 1 << 24
_FLOATS = {t: _lib.dtype_code(t) for t in (torch.bfloat16, torch.float16, torch.float32)}
INT8, E4M3, E4M3_GROUP = 1, 2, 3
GROUP = 128  # columns of an E4M3 group
ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}
_STEP = torch.tensor(1 / 127, dtype=torch.float32).item()


_no_gradients = _refusal("norms and products in 8 bits do")


def _padded(k: int) -> int:
    return -(-k // 128) * 128


def _storage_end(t: Tensor) -> int:
    """First address behind the storage of t."""
    s = t.untyped_storage()
    return s.data_ptr() + s.nbytes()


def _check_float(t: Tensor, name: str) -> None:
    if t.dtype not in _FLOATS:
        raise ValueError(f"{name} must be bf16, fp16 or fp32, got {t.dtype}")


def _flat(t: Tensor, name: str, cols: int | None = None) -> Tensor:
    """t [..., cols] as rows [rows, cols] with contiguous columns."""
    shape = t.shape
    if len(shape) < 1 or (cols is not None and shape[-1] != cols):
        raise ValueError(f"{name} must be [..., {cols if cols is not None else 'columns'}], got {list(shape)}")
    if t.dtype not in _FLOATS:
        _check_float(t, name)
    if len(shape) != 2:
        rows = 1
        for size in shape[:-1]:
            rows *= size
        t = t.reshape(rows, shape[-1])
        shape = t.shape
    down, across = t.stride()
    if (across != 1 and shape[1] > 1) or (0 < down < shape[1] and shape[0] > 1):
        t = t.contiguous()
    return t


def _desc(t: Tensor) -> _lib.Rows:
    return _lib.Rows(t.data_ptr(), t.stride(0), _FLOATS[t.dtype])


def _check_sizes(rows: int, cols: int) -> None:
    if rows > MAX_ROWS:
        raise ValueError(f"row count outside [0, {MAX_ROWS}]")
    if not 1 <= cols <= MAX_K:
        raise ValueError(f"column count outside [1, {MAX_K}]")


def _gpu(device: torch.device, t: Tensor) -> torch.device:
    if device.type != "cuda":
        _device_of(t)  # raises: there is no CPU path
    return device


def _status(device: torch.device) -> int:
    """Address of the device's status word, which a capture must not be the first to need: it would lie in the graph's memory."""
    if device not in _STATES and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the device's status word does not exist yet: run this call once eagerly before capturing it")
    return device_state(device).status.data_ptr()


def _same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device}")


class QuantRows:
    """Rows [rows, columns] in 8 bits: ``values`` int8 or float8_e4m3fn,
    ``scales`` fp32 [rows] or (E4M3) [rows, columns / 128].

    Rows that do not have a zero up to each multiple of 128 columns behind
    them, as the calls of this package write them, are copied once, when the
    object is made; later writes to ``values`` given do not reach the copy.
    """

    __slots__ = ("shape", "format", "device", "desc", "_held", "_values", "_scales")
    ndim = 2
    requires_grad = False

    def __init__(self, values: Tensor, scales: Tensor):
        if values.ndim != 2 or values.dtype not in (torch.int8, FP8_DTYPE):
            raise ValueError("values must be int8 or float8_e4m3fn [rows, columns]")
        rows, cols = values.shape
        _check_sizes(rows, cols)
        grouped = scales.ndim == 2
        if grouped and (values.dtype is torch.int8 or cols % GROUP):
            raise ValueError("scales of groups need E4M3 values and a multiple of 128 columns")
        if scales.dtype is not torch.float32 or scales.shape != ((rows, cols // GROUP) if grouped else (rows,)):
            raise ValueError("scales must be fp32 [rows] or, for E4M3, [rows, columns / 128]")
        if scales.device != values.device:
            raise ValueError("values and scales must share a device")
        if values.dtype is not torch.int8:
            _no_gradients("values", values)
        _no_gradients("scales", scales)
        stride = values.stride(0)
        if cols % GROUP or values.stride(1) != 1 or stride % 16 or not cols <= stride < 1 << 23 or values.data_ptr() % 16:
            held = torch.zeros((rows, _padded(cols)), dtype=torch.int8, device=values.device)
            held[:, :cols] = values.view(torch.int8)
            values = held.view(values.dtype)[:, :cols]
        scales = scales.contiguous()
        self._values, self._scales, self._held = values, scales, None
        self.shape, self.device = values.shape, values.device
        self.format = E4M3_GROUP if grouped else INT8 if values.dtype is torch.int8 else E4M3
        self.desc = _lib.QuantRowsDesc(values.data_ptr(), values.stride(0), scales.data_ptr(), self.format)

    @classmethod
    def _new(cls, rows: int, cols: int, fmt: int, device) -> QuantRows:
        """Rows for a call to write: one piece of memory, the scales behind the values."""
        self = cls.__new__(cls)
        width = _padded(cols)
        self._held = held = torch.empty(rows * (width + 4 * (cols // GROUP if fmt == E4M3_GROUP else 1)), dtype=torch.int8,
                                        device=device)
        self._values = self._scales = None
        self.shape, self.device, self.format = torch.Size((rows, cols)), device, fmt
        at = held.data_ptr()
        self.desc = _lib.QuantRowsDesc(at, width, at + rows * width, fmt)
        return self

    @property
    def values(self) -> Tensor:
        if self._values is None:
            rows, cols = self.shape
            width = _padded(cols)
            values = self._held[:rows * width].view(rows, width)[:, :cols]
            self._values = values if self.format == INT8 else values.view(FP8_DTYPE)
        return self._values

    @property
    def scales(self) -> Tensor:
        if self._scales is None:
            rows, cols = self.shape
            scales = self._held[rows * _padded(cols):].view(torch.float32)
            self._scales = scales.view(rows, cols // GROUP) if self.format == E4M3_GROUP else scales
        return self._scales

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> Tensor:
        """[rows, columns]: what the codes stand for, code * scale rounded to ``dtype``."""
        if dtype not in _FLOATS:
            raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
        device = self.device
        if device.type != "cuda":
            _device_of(self.values)
        rows, cols = self.shape
        out = torch.empty(self.shape, dtype=dtype, device=device)
        if rows:
            with _on(device):
                _lib.check(_lib.library().dmoe_rows8_read(
                    self.desc, rows, cols, _lib.Rows(out.data_ptr(), cols, _FLOATS[dtype]), _stream(device)))
        return out


def quantize_rows(x: Tensor) -> QuantRows:
    """Rows x [..., columns] as 8-bit integers with a scale a row:
    max(max |x|, 1e-12) times 1/127 as fp32 has it.  A row with an infinity or NaN gets codes of 0
    and a scale of NaN, and raises the device status bit."""
    _no_gradients("x", x)
    x = _flat(x, "x")
    rows, cols = x.shape
    _check_sizes(rows, cols)
    device = _gpu(x.device, x)
    q = QuantRows._new(rows, cols, INT8, device)
    if rows:
        with _on(device):
            _lib.check(_lib.library().dmoe_int8_quantize(_desc(x), rows, cols, q.desc,
                                                         _status(device), _stream(device)))
    return q


class Int8Weight:
    """Matrix [out, in] of 8-bit integers, ``values`` int8 [N, K], with a scale
    for each of its rows, ``scales`` fp32 [N] (or [N, 1]).

    Rows that are not 16-byte aligned with storage for whole 16 bytes (K not a
    multiple of 16, say) are copied once, when the object is made.
    """

    __slots__ = ("values", "scales", "shape", "device", "desc")

    def __init__(self, values: Tensor, scales: Tensor):
        if values.dtype is not torch.int8 or values.ndim != 2 or not values.numel():
            raise ValueError("INT8 weight values must be int8 [N, K]")
        self.shape = n, k = values.shape
        if k > MAX_K or n > MAX_ROWS:
            raise ValueError(f"INT8 weight outside [{MAX_ROWS}, {MAX_K}]")
        if scales.dtype is not torch.float32 or scales.shape not in ((n,), (n, 1)):
            raise ValueError("INT8 weight scales must be fp32 [N]")
        self.device = values.device
        if scales.device != self.device:
            raise ValueError("values and scales must share a device")
        if scales.requires_grad or _LEVEL._current_level >= 0:
            _no_gradients("scales", scales)
        width = (k + 15) // 16 * 16
        stride, across = values.stride()
        if n == 1:
            stride = max(stride, width)
        at = values.data_ptr()
        if (across != 1 and k > 1) or stride % 16 or at % 16 or not width <= stride < 1 << 23 \
                or (width > k and at + (n - 1) * stride + width > _storage_end(values)):
            held = torch.zeros((n, width), dtype=torch.int8, device=values.device)
            held[:, :k] = values
            values, stride, at = held[:, :k], width, held.data_ptr()
        if scales.ndim != 1 or not scales.is_contiguous():
            scales = scales.reshape(n).contiguous()
        self.values, self.scales = values, scales
        self.desc = _lib.Int8WeightDesc(at, stride, scales.data_ptr(), n, k)

    @classmethod
    def quantize(cls, weight: Tensor) -> Int8Weight:
        """The nearest 8-bit integers of a float matrix [N, K], with scales as rows have them:
        max(max |row|, 1e-12) times 1/127 as fp32 has it, on every device."""
        if weight.ndim != 2 or not weight.is_floating_point():
            raise ValueError("weight must be a float matrix [N, K]")
        w = weight.detach().double()
        scales = w.abs().amax(1).float().clamp(min=1e-12) * _STEP
        return cls((w / scales.double()[:, None]).round().clamp(-127, 127).to(torch.int8), scales)


def _input(x, k: int):
    """(descriptor of float rows, descriptor of rows in 8 bits, leading shape, row count, what they point into)."""
    if isinstance(x, QuantRows):
        if x.format != INT8:
            raise ValueError("x must be rows of 8-bit integers")
        rows, cols = x.shape
        if cols != k:
            raise ValueError(f"x must have {k} columns, got {cols}")
        return None, x.desc, x.shape[:1], rows, x
    flat = _flat(x, "x", k)
    rows = flat.shape[0]
    _check_sizes(rows, k)
    return _desc(flat), None, x.shape[:-1], rows, flat


def _out_dtype(x, dtype: torch.dtype | None, residual: Tensor | None) -> torch.dtype:
    if dtype is None:
        dtype = residual.dtype if residual is not None else torch.bfloat16 if isinstance(x, QuantRows) else x.dtype
    if dtype not in _FLOATS:
        raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    return dtype


def _residual(residual: Tensor, lead: torch.Size, cols: int, dtype: torch.dtype) -> Tensor:
    if residual.shape != (*lead, cols) or residual.dtype is not dtype:
        raise ValueError(f"residual must be {dtype} {[*lead, cols]}")
    return _flat(residual, "residual")


def int8_linear(x: Tensor | QuantRows, weight: Int8Weight, *, bias: Tensor | None = None, residual: Tensor | None = None,
                dtype: torch.dtype | None = None) -> Tensor:
    """[..., N] = x w^T (+ bias fp32 [N]) (+ residual [..., N]) in ``dtype``
    (default: the residual's, else x's, else bf16).  x [..., K] is quantized
    on the way, or ``QuantRows`` of 8-bit integers."""
    n, k = weight.shape
    dtype = _out_dtype(x, dtype, residual)
    _no_gradients("x bias residual", x, bias, residual)
    floats, quant, lead, rows, held = _input(x, k)
    device = _gpu(weight.device, weight.values)
    if x.device != device or bias is not None or residual is not None:
        _same_device(device, x=x, bias=bias, residual=residual)
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.shape != (n,):
            raise ValueError(f"bias must be fp32 [{n}]")
        bias = bias.contiguous()
    add = _residual(residual, lead, n, dtype) if residual is not None else None
    out = torch.empty((rows, n), dtype=dtype, device=device)
    if rows:
        lib = _lib.library()
        with _on(device):
            need = lib.dmoe_int8_linear_workspace_bytes(rows, n, k, quant is not None)
            scratch = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            _lib.check(lib.dmoe_int8_linear(
                floats, quant, rows, weight.desc, bias.data_ptr() if bias is not None else None,
                _desc(add) if add is not None else None, _lib.Rows(out.data_ptr(), n, _FLOATS[dtype]),
                scratch.data_ptr() if need else None, need, _status(device), _stream(device)))
    return out if len(lead) == 1 else out.reshape(*lead, n)


def int8_feed_forward(x: Tensor | QuantRows, gate_up: Int8Weight, down: Int8Weight, *, activation: str = "silu",
                      residual: Tensor | None = None, dtype: torch.dtype | None = None) -> Tensor:
    """[..., N] = (act(x gate^T) * (x up^T)) down^T (+ residual) in ``dtype``
    (default as ``int8_linear``'s): ``gate_up`` [2 * I, K] holds the gate rows,
    then the up rows, ``down`` is [N, I].  The hidden rows are rounded to
    ``dtype`` and then to 8-bit integers with a scale a row; ``activation`` is
    "silu" or "gelu_tanh".  ``gate_up`` is smaller than 2 GiB."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    (n, inter), (both, k) = down.shape, gate_up.shape
    if both != 2 * inter:
        raise ValueError(f"gate_up must be [{2 * inter}, K] for down [{n}, {inter}]")
    dtype = _out_dtype(x, dtype, residual)
    _no_gradients("x residual", x, residual)
    floats, quant, lead, rows, held = _input(x, k)
    device = _gpu(gate_up.device, gate_up.values)
    if x.device != device or down.device != device or residual is not None:
        _same_device(device, x=x, down=down, residual=residual)
    add = _residual(residual, lead, n, dtype) if residual is not None else None
    out = torch.empty((rows, n), dtype=dtype, device=device)
    if rows:
        lib, code = _lib.library(), _FLOATS[dtype]
        with _on(device):
            need = lib.dmoe_int8_feed_forward_workspace_bytes(rows, n, k, inter, code)
            scratch = torch.empty(need, dtype=torch.uint8, device=device)
            _lib.check(lib.dmoe_int8_feed_forward(
                floats, quant, rows, gate_up.desc, down.desc, act, _desc(add) if add is not None else None,
                _lib.Rows(out.data_ptr(), n, code), scratch.data_ptr(), need, _status(device),
                _stream(device)))
    return out if len(lead) == 1 else out.reshape(*lead, n)


class Int8Linear(HeldTypes):
    """Dense linear on 8-bit integers: ``weight`` int8 [N, K] with fp32
    ``scales`` [N] and an optional ``bias`` [N]; ``forward`` takes rows
    [..., K] or ``QuantRows`` (so one norm's output serves several), and
    ``dtype`` is what ``QuantRows`` give where the call does not say.  The
    buffer ``qweight`` has K rounded up to a multiple of 16.  Casts of the
    module (``half()``, ``to(dtype)``) move the buffers and leave their types."""

    _held = ("qweight", "scales", "bias")

    def __init__(self, weight: Tensor, scales: Tensor, bias: Tensor | None = None, *, device=None,
                 dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if dtype not in _FLOATS:
            raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
        self.dtype = dtype
        device = weight.device if device is None else torch.device(device)
        held = Int8Weight(weight.to(device), scales.to(device))
        self.out_features, self.in_features = held.shape
        # whole rows of storage, so that a call only describes them
        self.register_buffer("qweight", held.values.as_strided((held.shape[0], -(-held.shape[1] // 16) * 16),
                                                               (held.desc.row_stride, 1)))
        self.register_buffer("scales", held.scales)
        self.register_buffer("bias", bias.detach().to(device, torch.float32) if bias is not None else None)

    def _weight(self) -> Int8Weight:
        return Int8Weight(self.qweight[:, :self.in_features], self.scales)

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, *, device=None, dtype: torch.dtype = torch.bfloat16) -> Int8Linear:
        """The nearest 8-bit integers of a float linear."""
        held = Int8Weight.quantize(linear.weight)
        bias = linear.bias.detach().clone() if linear.bias is not None else None  # the linear keeps its own
        return cls(held.values, held.scales, bias, device=device, dtype=dtype)

    def forward(self, x: Tensor | QuantRows, *, residual: Tensor | None = None, dtype: torch.dtype | None = None) -> Tensor:
        if dtype is None and residual is None and isinstance(x, QuantRows):
            dtype = self.dtype
        return int8_linear(x, self._weight(), bias=self.bias, residual=residual, dtype=dtype)


class Int8FeedForward(torch.nn.Module):
    """Gated feed-forward block on 8-bit integers: ``gate_up`` int8 [2 * I, K]
    (gate rows first), ``down`` int8 [N, I], each with its fp32 scales; ``dtype``
    as ``Int8Linear``'s."""

    def __init__(self, gate_up: Tensor, gate_up_scales: Tensor, down: Tensor, down_scales: Tensor, *,
                 activation: str = "silu", device=None, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
        if gate_up.ndim != 2 or down.ndim != 2 or gate_up.shape[0] != 2 * down.shape[1]:
            raise ValueError("gate_up must be [2 * I, K] for down [N, I]")
        self.activation = activation
        self.gate_up = Int8Linear(gate_up, gate_up_scales, device=device, dtype=dtype)
        self.down = Int8Linear(down, down_scales, device=device, dtype=dtype)

    @classmethod
    def from_linears(cls, gate: torch.nn.Linear, up: torch.nn.Linear, down: torch.nn.Linear, *, activation: str = "silu",
                     device=None, dtype: torch.dtype = torch.bfloat16) -> Int8FeedForward:
        """The nearest 8-bit integers of a float block's three linears, which have no bias."""
        if any(linear.bias is not None for linear in (gate, up, down)):
            raise ValueError("the linears of a gated feed-forward block have no bias here")
        w, v = Int8Weight.quantize(torch.cat([gate.weight, up.weight])), Int8Weight.quantize(down.weight)
        return cls(w.values, w.scales, v.values, v.scales, activation=activation, device=device, dtype=dtype)

    def forward(self, x: Tensor | QuantRows, *, residual: Tensor | None = None, dtype: torch.dtype | None = None) -> Tensor:
        if dtype is None and residual is None and isinstance(x, QuantRows):
            dtype = self.down.dtype
        return int8_feed_forward(x, self.gate_up._weight(), self.down._weight(), activation=self.activation,
                                 residual=residual, dtype=dtype)
