"""Attention over a key/value cache held in 4 bits.

``KvCache4`` is a paged cache of 4.5 bits a value (codes and scale words,
layout in include/drama_moe.h).  ``append`` rotates queries and keys by their
positions (``Rotary``: one axis, or several, as time / height / width) and
quantizes keys and values into the pages; ``attend`` is causal attention of
the same rows over what the pages hold, for one new token a sequence as for
whole prompts; ``read`` brings the held values back.  ``PagedBatch`` says
which rows belong to which sequence and where its pages are.

The reference leaves attention to the model it drives, with a bf16 cache of
``sequence_capacity`` tokens (src/drama_low_vram/backbone_graph.py:123-128).
No call synchronizes the host, every call can be captured in a hipGraph, and
scratch is allocated for each call by torch, so calls on several streams and
graphs captured apart share nothing but the cache and the status word.  There is
no backward: with gradients enabled, inputs that need them are refused.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _lib
from .offload import _device_of, device_state

GROUP = 32            # channels a scale word
MAX_SEQUENCES = 4096
MAX_ROWS = 1 << 24
_HALVES = (torch.bfloat16, torch.float16)


def _rows(t: Tensor, name: str, shape: tuple, dtype: torch.dtype | None, device, *, written: bool = False):
    """t as rows of ``shape`` [rows, heads, dim] with contiguous, 16-byte
    aligned heads -- itself, or (for one that is only read) a copy -- and its
    descriptor."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype not in _HALVES:
        raise ValueError(f"{name} must be bf16 or fp16, got {t.dtype}")
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    s0, s1, s2 = t.stride()
    rows, heads = shape[0] > 1, shape[1] > 1
    address = t.data_ptr()
    if s2 != 1 or (s0 % 8 and rows) or (s1 % 8 and heads) or address % 16:
        if written:
            raise ValueError(f"{name} must have contiguous, 16-byte aligned heads")
        t = t.clone(memory_format=torch.contiguous_format)
        (s0, s1, _), address = t.stride(), t.data_ptr()
    # a dimension of one entry has no stride
    return t, _lib.HeadRows(address, s0 if rows else 0, s1 if heads else 0)


def _new(shape: tuple, dtype: torch.dtype, device):
    """New rows of ``shape`` and their descriptor."""
    t = torch.empty(shape, dtype=dtype, device=device)
    rows, heads, dim = shape
    return t, _lib.HeadRows(t.data_ptr(), heads * dim if rows > 1 else 0, dim if heads > 1 else 0)


def _no_gradients(names: str, *tensors: Tensor | None) -> None:
    """Refuses inputs whose gradients the kernels, which have no backward, would lose."""
    if torch.is_grad_enabled():
        for i, t in enumerate(tensors):
            if t is not None and t.requires_grad:
                raise ValueError(f"{names.split()[i]} needs gradients, which attention over the cache does not have: "
                                 "call it under torch.no_grad()")


def _heads(q: Tensor) -> int:
    return q.shape[1] if q.ndim == 3 else 0


def _indices(t: Tensor, name: str, ndim: int) -> Tensor:
    if t.dtype is not torch.int32 or t.ndim != ndim or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be int32 with {ndim} dimension(s) and contiguous rows")
    return t


class PagedBatch:
    """Rows of a call over paged sequences.

    ``block_table`` [S, pages] int32 names the pages of each sequence's
    tokens (sequences on the same pages may share a row: ``row.expand(S, -1)``), ``lengths`` [S] int32 counts its tokens with the call's rows among
    them, and ``starts`` [S + 1] int32 are the offsets of each sequence's rows
    in the row buffers, which must not decrease (None: row s is sequence s).  With n rows, a
    sequence's rows are its last n tokens.  ``rows`` is the row count of the
    buffers and ``max_rows`` the most rows a sequence has (default: ``rows``;
    1 without ``starts``).  The three tables stay the caller's: their contents
    may change between calls and between replays of a captured call.  Rows
    that no sequence owns -- behind the last one -- are left as they are.
    ``max_rows`` picks the attention kernel for all sequences: a prompt and
    single tokens are better attended as two batches.
    """

    __slots__ = ("block_table", "lengths", "starts", "rows", "max_rows", "desc", "device", "scratch")

    def __init__(self, block_table: Tensor, lengths: Tensor, starts: Tensor | None = None, *, rows: int | None = None,
                 max_rows: int | None = None):
        _indices(block_table, "block_table", 2)
        _indices(lengths, "lengths", 1)
        seqs, cols = block_table.shape
        if lengths.shape[0] != seqs:
            raise ValueError("block_table and lengths must have one entry a sequence")
        if not 1 <= seqs <= MAX_SEQUENCES:
            raise ValueError(f"sequence count outside [1, {MAX_SEQUENCES}]")
        if cols < 1:
            raise ValueError("block_table has no pages")
        # sequences on the same pages may share one row of the table (stride 0)
        stride = block_table.stride(0) if seqs > 1 else cols
        if 0 < stride < cols:
            raise ValueError("block_table rows overlap")
        device = lengths.device
        if block_table.device != device:
            raise ValueError("batch tables must share a device")
        if starts is not None:
            _indices(starts, "starts", 1)
            if starts.shape[0] != seqs + 1:
                raise ValueError("starts must be [sequences + 1]")
            if starts.device != device:
                raise ValueError("batch tables must share a device")
            if rows is None:
                raise ValueError("rows is required with starts")
            rows = int(rows)
            max_rows = rows if max_rows is None else int(max_rows)
            if rows < 0:
                raise ValueError("rows must not be negative")
        else:
            rows = seqs if rows is None else int(rows)
            max_rows = 1 if max_rows is None else int(max_rows)
            if rows < seqs:
                raise ValueError("rows must cover every sequence")
        if rows > MAX_ROWS:  # the descriptor has 32 bits for it
            raise ValueError(f"row count outside [0, {MAX_ROWS}]")
        if rows and not 1 <= max_rows <= rows:
            raise ValueError("max_rows outside [1, rows]")
        self.block_table, self.lengths, self.starts = block_table, lengths, starts
        self.rows, self.max_rows, self.device = rows, max_rows, device
        self.scratch = {}  # bytes that attention over this batch's sizes needs, by geometry
        self.desc = _lib.Kv4Batch(block_table.data_ptr(), stride, lengths.data_ptr(),
                                  starts.data_ptr() if starts is not None else None, seqs, cols, rows, max_rows)


class Rotary:
    """Rotation of the first 2 * len(inv_freq) channels of a head by position.

    Pair i -- channels (i, i + R/2) of R, or (2i, 2i + 1) with ``interleaved``
    -- turns by ``position * inv_freq[i]``, where the position is that of
    axis ``axis[i]`` (uint8 [R/2]; None: the first), the last one where there
    are fewer.  ``sections`` makes such an axis table from frequency counts.
    Angles are formed in 64 bits.
    """

    __slots__ = ("inv_freq", "axis", "dim", "interleaved")

    def __init__(self, inv_freq: Tensor, *, axis: Tensor | None = None, interleaved: bool = False):
        if inv_freq.dtype != torch.float32 or inv_freq.ndim != 1 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous fp32 [R/2]")
        if inv_freq.shape[0] < 8 or inv_freq.shape[0] % 8:
            raise ValueError("the rotated channels must be a multiple of 16")
        if axis is not None and (axis.dtype != torch.uint8 or axis.shape != inv_freq.shape or not axis.is_contiguous()
                                 or axis.device != inv_freq.device):
            raise ValueError("axis must be contiguous uint8 [R/2] on inv_freq's device")
        self.inv_freq, self.axis = inv_freq, axis
        self.dim, self.interleaved = 2 * inv_freq.shape[0], bool(interleaved)

    @staticmethod
    def sections(counts, *, cyclic: bool = False, device=None) -> Tensor:
        """Axis table of frequency counts a axis: the axes one after the other,
        or (``cyclic``) in turn as long as each has frequencies left."""
        counts = [int(c) for c in counts]
        if not counts or min(counts) < 0 or len(counts) > 255:
            raise ValueError("sections needs the frequency count of each axis")
        if not cyclic:
            table = [a for a, c in enumerate(counts) for _ in range(c)]
        else:
            left, table = list(counts), []
            while any(left):
                for a, c in enumerate(left):
                    if c:
                        table.append(a)
                        left[a] -= 1
        return torch.tensor(table, dtype=torch.uint8, device=device)


class KvCache4:
    """Paged key/value cache of 4-bit codes over ``pages`` uint8 [num_pages,
    kv_heads, page_size * (D + D/8)] (pages may be strided, as in a buffer
    that holds several layers')."""

    __slots__ = ("pages", "page_size", "kv_heads", "head_dim", "desc", "device", "_state", "_status")

    def __init__(self, pages: Tensor, *, page_size: int, head_dim: int):
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size must be a power of two in [16, 256]")
        need = self.head_bytes(page_size, head_dim)
        if pages.dtype != torch.uint8 or pages.ndim != 3 or pages.shape[2] != need or not pages.numel():
            raise ValueError(f"pages must be uint8 [num_pages, kv_heads, {need}]")
        stride = pages.stride(0) if pages.shape[0] > 1 else max(pages.stride(0), pages.shape[1] * need)
        if pages.stride(2) != 1 or (pages.shape[1] > 1 and pages.stride(1) != need) or stride % 16 \
                or pages.data_ptr() % 16:
            raise ValueError("a page must be contiguous and 16-byte aligned")
        self.pages, self.page_size, self.head_dim = pages, page_size, head_dim
        self.kv_heads = pages.shape[1]
        self.device = pages.device
        # the device's status word, made here and never inside a capture
        self._state = device_state(pages.device) if pages.is_cuda else None
        self._status = self._state.status.data_ptr() if pages.is_cuda else None
        self.desc = _lib.Kv4Cache(pages.data_ptr(), stride, pages.shape[0], page_size, self.kv_heads, head_dim)

    @staticmethod
    def head_bytes(page_size: int, head_dim: int) -> int:
        """Bytes of one head's part of a page."""
        return page_size * (head_dim + head_dim // 8)

    @classmethod
    def allocate(cls, num_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, device=None) -> KvCache4:
        """A cache of zeroed pages."""
        pages = torch.zeros((num_pages, kv_heads, cls.head_bytes(page_size, head_dim)), dtype=torch.uint8, device=device)
        return cls(pages, page_size=page_size, head_dim=head_dim)

    def _check(self, batch: PagedBatch) -> torch.device:
        if self._state is None:
            _device_of(self.pages)  # raises: there is no CPU path
        if batch.device != self.device:
            raise ValueError("cache and batch must share a device")
        return self.device

    def status(self, clear: bool = True) -> int:
        """Read (and clear) the device status bits; synchronizes the stream."""
        if self._state is None:
            _device_of(self.pages)
        value = int(self._state.status.item())
        if clear:
            self._state.status.zero_()
        return value

    def append(self, k: Tensor, v: Tensor, batch: PagedBatch, *, rotary: Rotary | None = None,
               positions: Tensor | None = None, q: Tensor | None = None, q_out: Tensor | None = None) -> Tensor | None:
        """Stores keys and values [rows, kv_heads, D] of the batch's rows, keys
        rotated.  ``positions`` is int32 or int64 [rows] or [axes, rows]
        (None: places in the sequences).  With ``q`` [rows, heads, D] returns
        its rotation, in ``q_out`` if given (which may be ``q``)."""
        device = self._check(batch)
        rows, dim = batch.rows, self.head_dim
        dtype = k.dtype
        shape = (rows, self.kv_heads, dim)
        k, k_rows = _rows(k, "k", shape, None, device)
        v, v_rows = _rows(v, "v", shape, dtype, device)
        heads, q_rows, out_rows = 0, None, None
        if q is not None:
            heads = _heads(q)
            shape = (rows, heads, dim)
            q, q_rows = _rows(q, "q", shape, dtype, device)
            if q_out is None:
                q_out, out_rows = _new(shape, dtype, device)
            else:
                _, out_rows = _rows(q_out, "q_out", shape, dtype, device, written=True)
        elif q_out is not None:
            raise ValueError("q_out needs q")
        turn = None
        if rotary is not None:
            if rotary.dim > dim:
                raise ValueError("more rotated channels than head_dim")
            if rotary.inv_freq.device != device:
                raise ValueError("rotary and cache must share a device")
            axes, stride = 1, 0
            if positions is not None:
                if positions.dtype not in (torch.int32, torch.int64) or positions.ndim not in (1, 2) \
                        or positions.shape[-1] != rows:
                    raise ValueError("positions must be int32 or int64 [rows] or [axes, rows]")
                if positions.device != device:
                    raise ValueError("positions must be on the cache's device")
                if rows and (positions.stride(-1) != 1 or (positions.ndim == 2 and positions.stride(0) < rows)):
                    positions = positions.contiguous()
                if positions.ndim == 2:
                    axes, stride = positions.shape[0], positions.stride(0)
                if not axes:
                    raise ValueError("positions has no axis")
            turn = _lib.RotaryDesc(
                rotary.inv_freq.data_ptr(), rotary.axis.data_ptr() if rotary.axis is not None else None,
                positions.data_ptr() if positions is not None else None, stride,
                _lib.I32 if positions is not None and positions.dtype == torch.int32 else _lib.I64, axes, rotary.dim,
                int(rotary.interleaved))
        elif positions is not None:
            raise ValueError("positions need a rotary")
        _no_gradients("k v q q_out", k, v, q, q_out)
        if rows == 0:
            return q_out
        with _on(device):
            _lib.check(_lib.library().dmoe_kv4_append(
                self.desc, batch.desc, turn, q_rows, heads, out_rows, k_rows, v_rows, _lib.dtype_code(dtype), self._status, _stream(device)))
        return q_out

    def read(self, batch: PagedBatch, *, dtype: torch.dtype = torch.float16, k_out: Tensor | None = None,
             v_out: Tensor | None = None):
        """(keys, values) [rows, kv_heads, D] that the cache holds for the
        batch's rows: keys as rotated, exact in fp16."""
        device = self._check(batch)
        shape = (batch.rows, self.kv_heads, self.head_dim)
        if dtype not in _HALVES:
            raise ValueError(f"k_out must be bf16 or fp16, got {dtype}")
        k_out, k_rows = _new(shape, dtype, device) if k_out is None else _rows(k_out, "k_out", shape, dtype, device,
                                                                               written=True)
        v_out, v_rows = _new(shape, dtype, device) if v_out is None else _rows(v_out, "v_out", shape, dtype, device,
                                                                               written=True)
        _no_gradients("k_out v_out", k_out, v_out)
        if batch.rows:
            with _on(device):
                _lib.check(_lib.library().dmoe_kv4_read(
                    self.desc, batch.desc, k_rows, v_rows, _lib.dtype_code(dtype), self._status, _stream(device)))
        return k_out, v_out

    def attend(self, q: Tensor, batch: PagedBatch, *, scale: float | None = None, window: int = 0,
               out: Tensor | None = None) -> Tensor:
        """Attention of queries [rows, heads, D] over the cache: a row sees the
        tokens up to its own place, with ``window`` only that many of them; one
        that sees none becomes 0.  Table entries behind the windows of all rows
        may name no page.  ``scale`` defaults to D ** -0.5.  Rows that
        no sequence owns are not written (in a new ``out`` they hold nothing)."""
        device = self._check(batch)
        heads = _heads(q)
        shape = (batch.rows, heads, self.head_dim)
        q, q_rows = _rows(q, "q", shape, None, device)
        if heads < 1 or heads % self.kv_heads:
            raise ValueError("query heads must be a multiple of the key/value heads")
        if not -2 ** 31 <= window < 2 ** 31:
            raise ValueError("window must fit 32 bits")
        _no_gradients("q out", q, out)
        if out is None:
            out, out_rows = _new(shape, q.dtype, device)
        else:
            _, out_rows = _rows(out, "out", shape, q.dtype, device, written=True)
        if batch.rows == 0:
            return out
        lib = _lib.library()
        with _on(device):
            need = batch.scratch.get((heads, self.kv_heads, self.head_dim, self.page_size))
            if need is None:
                need = lib.dmoe_kv4_attention_workspace_bytes(self.desc, batch.desc, heads)
                batch.scratch[heads, self.kv_heads, self.head_dim, self.page_size] = need
            scratch = torch.empty(need, dtype=torch.uint8, device=device)
            _lib.check(lib.dmoe_kv4_attention(
                self.desc, batch.desc, q_rows, heads, self.head_dim ** -0.5 if scale is None else scale, window,
                out_rows, _lib.dtype_code(q.dtype), scratch.data_ptr(), need, self._status, _stream(device)))
        return out


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _on(device: torch.device):
    """The launches of a call go to its tensors' device, whichever is current."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    """hipStream_t of torch's current stream on ``device``."""
    return torch._C._cuda_getCurrentRawStream(device.index)
