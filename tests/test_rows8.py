"""Rows and products in 8 bits on the CPU: refusals of the Python and C entry
points before any launch, the copies that misaligned operands get, and
properties of the reference that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

import rows8_reference as ref
from drama_moe import _lib, int8
from drama_moe.attention import KvCache4, PagedBatch
from drama_moe.block import AttentionBlock, DenseBlock
from drama_moe.int8 import (Int8FeedForward, Int8Linear, Int8Weight, QuantRows, int8_feed_forward, int8_linear,
                            quantize_rows)
from drama_moe.norm import RmsNorm, rms_norm

BF16, F32 = torch.bfloat16, torch.float32


def i8(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def weight(n=4, k=32):
    return Int8Weight(i8(n, k) + 1, torch.ones(n))


@pytest.mark.parametrize("make,message", [
    (lambda: QuantRows(torch.zeros(2, 32), torch.ones(2)), "int8 or float8_e4m3fn"),
    (lambda: QuantRows(i8(2, 2, 32), torch.ones(2)), "int8 or float8_e4m3fn"),
    (lambda: QuantRows(i8(2, 32), torch.ones(3)), "scales must be fp32"),
    (lambda: QuantRows(i8(2, 32), torch.ones(2).double()), "scales must be fp32"),
    (lambda: QuantRows(i8(2, 256), torch.ones(2, 2)), "groups need E4M3"),
    (lambda: QuantRows(i8(2, 130).view(torch.float8_e4m3fn), torch.ones(2, 1)), "groups need E4M3"),
    (lambda: QuantRows(i8(2, 256).view(torch.float8_e4m3fn), torch.ones(2, 1)), "scales must be fp32"),
    (lambda: QuantRows(i8(2, 0), torch.ones(2)), "column count outside"),
    (lambda: QuantRows(i8(1, 65537), torch.ones(1)), "column count outside"),
    (lambda: QuantRows(i8(2, 32), torch.ones(2)).dequantize(torch.int8), "dtype must be"),
    (lambda: quantize_rows(torch.zeros(2, 32).double()), "x must be bf16, fp16 or fp32"),
    (lambda: quantize_rows(torch.zeros(2, 0)), "column count outside"),
    (lambda: quantize_rows(torch.zeros(2, 32, requires_grad=True)), "x needs gradients"),
    (lambda: Int8Weight(torch.zeros(4, 32), torch.ones(4)), "int8 \\[N, K\\]"),
    (lambda: Int8Weight(i8(0, 32), torch.ones(0)), "int8 \\[N, K\\]"),
    (lambda: Int8Weight(i8(4, 32), torch.ones(5)), "scales must be fp32 \\[N\\]"),
    (lambda: Int8Weight(i8(4, 32), torch.ones(2, 2)), "scales must be fp32 \\[N\\]"),
    (lambda: Int8Weight(i8(4, 32), torch.ones(4).half()), "scales must be fp32 \\[N\\]"),
    (lambda: Int8Weight(i8(1, 65537), torch.ones(1)), "weight outside"),
    (lambda: Int8Weight.quantize(i8(2, 2)), "float matrix"),
    (lambda: int8_linear(torch.zeros(2, 31), weight()), "x must be \\[..., 32\\]"),
    (lambda: int8_linear(torch.zeros(2, 32).double(), weight()), "dtype must be"),
    (lambda: int8_linear(torch.zeros(2, 32).double(), weight(), dtype=F32), "x must be bf16, fp16 or fp32"),
    (lambda: int8_linear(QuantRows(i8(2, 48), torch.ones(2)), weight()), "x must have 32 columns"),
    (lambda: int8_linear(QuantRows(i8(2, 32).view(torch.float8_e4m3fn), torch.ones(2)), weight()), "8-bit integers"),
    (lambda: int8_linear(torch.zeros(2, 32), weight(), dtype=torch.int32), "dtype must be"),
    (lambda: int8_linear(torch.zeros(2, 32, requires_grad=True), weight()), "x needs gradients"),
    (lambda: int8_linear(torch.zeros(2, 32), weight(), bias=torch.zeros(4, requires_grad=True)), "bias needs gradients"),
    (lambda: int8_feed_forward(torch.zeros(2, 32), weight(8), weight(5, 4), activation="relu"), "activation must be"),
    (lambda: int8_feed_forward(torch.zeros(2, 32), weight(8), weight(5, 3)), "gate_up must be \\[6, K\\]"),
    (lambda: int8_feed_forward(torch.zeros(2, 16), weight(8), weight(5, 4)), "x must be \\[..., 32\\]"),
    (lambda: int8_feed_forward(torch.zeros(2, 32), weight(8), weight(5, 4),
                               residual=torch.zeros(2, 5, requires_grad=True)), "residual needs gradients"),
    (lambda: Int8FeedForward(i8(8, 32), torch.ones(8), i8(5, 3), torch.ones(5)), "gate_up must be"),
    (lambda: Int8FeedForward(i8(8, 32), torch.ones(8), i8(5, 4), torch.ones(5), activation="relu"), "activation must be"),
    (lambda: Int8FeedForward.from_linears(*(torch.nn.Linear(8, 8) for _ in range(3))), "have no bias"),
    (lambda: rms_norm(torch.zeros(2, 32), torch.ones(31)), "weight must be \\[32\\]"),
    (lambda: rms_norm(torch.zeros(2, 32), torch.ones(32).int()), "weight must be bf16"),
    (lambda: rms_norm(torch.zeros(2, 32).int(), torch.ones(32)), "x must be bf16"),
    (lambda: rms_norm(torch.zeros(2, 32), torch.ones(32), quant="int4"), "quant must be one of"),
    (lambda: rms_norm(torch.zeros(2, 32), torch.ones(32), quant="fp8-128"), "multiple of 128"),
    (lambda: rms_norm(torch.zeros(2, 32), torch.ones(32), rows=False), "no output"),
    (lambda: rms_norm(torch.zeros(2, 32), torch.ones(32), residual=torch.zeros(1, 32)), "residual must be"),
    (lambda: rms_norm(torch.zeros(2, 32), torch.ones(32), residual=torch.zeros(2, 32).half()), "residual must be"),
    (lambda: rms_norm(torch.zeros(2, 32), torch.ones(32, requires_grad=True)), "weight needs gradients"),
    (lambda: rms_norm(torch.zeros(1, 65537), torch.ones(65537)), "column count outside"),
    (lambda: RmsNorm(torch.ones(2, 2)), "weight must be \\[columns\\]"),
    (lambda: RmsNorm(torch.ones(2), quant="int4"), "quant must be one of"),
])
def test_refusals(make, message):
    with pytest.raises(ValueError, match=message):
        make()


@pytest.mark.parametrize("call", [
    lambda: quantize_rows(torch.zeros(2, 32)), lambda: QuantRows(i8(2, 32), torch.ones(2)).dequantize(),
    lambda: int8_linear(torch.zeros(2, 32), weight()), lambda: int8_feed_forward(torch.zeros(2, 32), weight(8), weight(5, 4)),
    lambda: rms_norm(torch.zeros(2, 32), torch.ones(32)),
    lambda: Int8Linear(i8(4, 32), torch.ones(4))(torch.zeros(2, 32)),
])
def test_there_is_no_cpu_path(call):
    with pytest.raises(RuntimeError, match="requires tensors on a ROCm GPU"):
        call()


def test_residual_and_bias_shapes():
    w = weight()
    with pytest.raises((ValueError, RuntimeError)):
        int8_linear(torch.zeros(2, 32), w, bias=torch.zeros(3))
    # on the CPU the device is refused first; the shapes by themselves:
    from drama_moe.int8 import _residual
    for bad in (torch.zeros(2, 5), torch.zeros(3, 4), torch.zeros(2, 4).half(), torch.zeros(4)):
        with pytest.raises(ValueError, match="residual must be"):
            _residual(bad, torch.Size([2]), 4, F32)
    assert _residual(torch.zeros(3, 2, 4), torch.Size([3, 2]), 4, F32).shape == (6, 4)


def test_rows_are_held_with_their_zeros():
    """Widths that are no multiple of 128 are copied, others stay where they are if a call can read them there."""
    x = torch.arange(1, 41, dtype=torch.int8).reshape(2, 20)
    q = QuantRows(x, torch.ones(2))
    assert q.shape == (2, 20) and torch.equal(q.values, x) and q.values.stride() == (128, 1)
    assert not q.values.as_strided((2, 128), (128, 1))[:, 20:].any()
    big = i8(4, 512)
    assert QuantRows(big, torch.ones(4)).values.data_ptr() == big.data_ptr()
    assert QuantRows(big[:, 128:384], torch.ones(4)).desc.row_stride == 512
    for apart in (big[:, 1:257], big.t().contiguous().t()[:, :256], big[:1, :256].expand(4, 256)):
        q = QuantRows(apart, torch.ones(4))
        assert q.desc.row_stride == 256 and torch.equal(q.values, apart)
    e = torch.zeros(2, 20).to(torch.float8_e4m3fn)
    assert QuantRows(e, torch.ones(2)).values.dtype == torch.float8_e4m3fn
    made = QuantRows._new(3, 200, 1, torch.device("cpu"))
    assert made.shape == (3, 200) and made.values.stride() == (256, 1) and made.scales.shape == (3,)
    assert QuantRows._new(3, 256, 3, torch.device("cpu")).scales.shape == (3, 2)


def test_matrices_are_read_where_they_lie():
    big = i8(10, 320)
    for w in (big, big[:, :300], big[2:7, 16:300], big[::2]):
        held = Int8Weight(w, torch.ones(w.shape[0], 1))
        assert held.values.data_ptr() == w.data_ptr() and held.desc.row_stride == w.stride(0)
    last = i8(10 * 320 - 1)  # the last row's storage ends inside its last sixteen bytes
    w = last.as_strided((10, 319), (320, 1))
    assert Int8Weight(w, torch.ones(10)).values.data_ptr() != w.data_ptr()
    for w in (big[:, 1:300], big.t(), i8(5, 33), big[:1].expand(5, 320)):
        held = Int8Weight(w, torch.ones(w.shape[0]))
        assert held.values.data_ptr() != w.data_ptr() and torch.equal(held.values, w)
        assert held.desc.row_stride == -(-w.shape[1] // 16) * 16 and (held.desc.n, held.desc.k) == w.shape
    one = i8(33)[None]  # one row: its stride does not matter, its storage does
    assert Int8Weight(one, torch.ones(1)).values.data_ptr() != one.data_ptr()
    assert Int8Weight(i8(48)[None, :33], torch.ones(1)).desc.row_stride == 48


def test_nearest_integers_of_a_float_matrix():
    torch.manual_seed(0)
    w = torch.randn(20, 70)
    w[3] = 0
    held = Int8Weight.quantize(w)
    assert (held.values[3] == 0).all()
    assert ((held.values.double() * held.scales.double()[:, None] - w.double()).abs() <= held.scales.double()[:, None] * 0.5000001).all()


# ------------------------------------------------------------------ C entry points

def rows(data=0x100000, stride=256, dtype=_lib.F32):
    return _lib.Rows(data, stride, dtype)


def q8(values=0x200000, stride=256, scales=0x300000, fmt=1):
    return _lib.QuantRowsDesc(values, stride, scales, fmt)


def w8(values=0x400000, stride=256, scales=0x500000, n=64, k=256):
    return _lib.Int8WeightDesc(values, stride, scales, n, k)


P = ctypes.c_void_p


def norm(x=rows(), residual=None, count=4, cols=256, weight=P(0x600000), wdtype=_lib.F32, offset=0.0, eps=1e-6, hidden=None,
         out=rows(), quant=None):
    return _lib.library().dmoe_rms_norm(x, residual, count, cols, weight, wdtype, offset, eps, hidden, out, quant, None, None)


def linear(x=None, quant=q8(), count=4, w=w8(), bias=None, residual=None, out=rows(), ws=None, ws_bytes=0):
    return _lib.library().dmoe_int8_linear(x, quant, count, w, bias, residual, out, ws, ws_bytes, None, None)


def ffn(x=None, quant=q8(), count=4, up=w8(n=128), down=w8(n=256, k=64), act=0, residual=None, out=rows(), ws=P(0x700000),
        ws_bytes=1 << 20):
    return _lib.library().dmoe_int8_feed_forward(x, quant, count, up, down, act, residual, out, ws, ws_bytes, None, None)


@pytest.mark.parametrize("call,message", [
    (lambda: norm(x=None), "x rows are required"),
    (lambda: norm(x=rows(data=0x100002)), "aligned to its elements"),
    (lambda: norm(x=rows(dtype=_lib.I32)), "must be fp32, bf16 or fp16"),
    (lambda: norm(x=rows(stride=255)), "row stride out of range"),
    (lambda: norm(x=rows(stride=-256)), "row stride out of range"),
    (lambda: norm(x=rows(stride=1 << 40)), "row stride out of range"),
    (lambda: norm(count=-1), "row count outside"),
    (lambda: norm(count=(1 << 24) + 1), "row count outside"),
    (lambda: norm(cols=0), "column count outside"),
    (lambda: norm(cols=65537), "column count outside"),
    (lambda: norm(weight=None), "norm weight"),
    (lambda: norm(weight=P(0x600001)), "aligned to its elements"),
    (lambda: norm(eps=-1.0), "eps not negative"),
    (lambda: norm(eps=float("nan")), "eps not negative"),
    (lambda: norm(offset=float("inf")), "must be finite"),
    (lambda: norm(out=None), "no output"),
    (lambda: norm(hidden=rows()), "need a residual"),
    (lambda: norm(residual=rows(dtype=_lib.F16)), "residual must have the type"),
    (lambda: norm(residual=rows(), hidden=rows(dtype=_lib.F16)), "hidden must have the type"),
    (lambda: norm(out=rows(dtype=_lib.F16)), "out must have the type"),
    (lambda: norm(out=rows(stride=0)), "row stride out of range"),
    (lambda: norm(quant=q8(fmt=0)), "unknown format"),
    (lambda: norm(quant=q8(fmt=4)), "unknown format"),
    (lambda: norm(quant=q8(values=0x200008)), "16-byte aligned"),
    (lambda: norm(quant=q8(scales=None)), "are required"),
    (lambda: norm(quant=q8(stride=240)), "row stride"),
    (lambda: norm(cols=250, quant=q8(stride=250)), "row stride"),
    (lambda: norm(quant=q8(stride=1 << 23)), "row stride"),
    (lambda: norm(cols=200, quant=q8(fmt=3)), "multiple of 128"),
    (lambda: _lib.library().dmoe_int8_quantize(rows(), 4, 256, q8(fmt=2), None, None), "8-bit integers"),
    (lambda: _lib.library().dmoe_int8_quantize(None, 4, 256, q8(), None, None), "x rows are required"),
    (lambda: _lib.library().dmoe_rows8_read(q8(), 4, 256, None, None), "out rows are required"),
    (lambda: _lib.library().dmoe_rows8_read(None, 4, 256, rows(), None), "are required"),
    (lambda: linear(quant=None), "either quantized or not"),
    (lambda: linear(x=rows()), "either quantized or not"),
    (lambda: linear(w=None), "INT8 weight"),
    (lambda: linear(w=w8(values=0x400004)), "16-byte aligned"),
    (lambda: linear(w=w8(stride=255)), "row stride"),
    (lambda: linear(w=w8(stride=1 << 23)), "row stride"),
    (lambda: linear(w=w8(n=0)), "weight rows outside"),
    (lambda: linear(w=w8(k=65537)), "weight columns outside"),
    (lambda: linear(quant=q8(fmt=2)), "8-bit integers"),
    (lambda: linear(quant=q8(stride=128)), "row stride"),
    (lambda: linear(out=rows(stride=63)), "out has a row stride"),
    (lambda: linear(bias=P(0x800002)), "bias must be aligned"),
    (lambda: linear(residual=rows(dtype=_lib.BF16)), "residual must have the type"),
    (lambda: linear(x=rows(), quant=None, count=100), "workspace too small"),
    (lambda: linear(x=rows(), quant=None, count=100, ws=P(0x700010), ws_bytes=1 << 20), "256-byte aligned"),
    (lambda: ffn(down=w8(n=256, k=63)), "gate_up must be"),
    (lambda: ffn(up=w8(n=129)), "gate_up must be"),
    (lambda: ffn(act=2), "unknown activation"),
    (lambda: ffn(ws_bytes=100), "workspace too small"),
    (lambda: ffn(ws=None), "workspace too small"),
    (lambda: ffn(x=rows()), "either quantized or not"),
    (lambda: ffn(up=w8(n=1 << 16, stride=1 << 15), down=w8(n=256, k=1 << 15, stride=1 << 15)), "smaller than 2 GiB"),
])
def test_entry_points_refuse(call, message):
    assert call() == -1
    assert message in _lib.library().dmoe_last_error().decode()


def test_workspaces_cover_what_calls_hold():
    lib = _lib.library()
    for count, k in ((17, 1 << 16), (5, 100), (65, 4096), (1 << 24, 65536)):
        need = lib.dmoe_int8_linear_workspace_bytes(count, 512, k, 0)
        assert need >= count * (-(-k // 128) * 128 + 4) and need % 32 == 0
        assert need > lib.dmoe_int8_linear_workspace_bytes(count, 512, k, 1)
        both = lib.dmoe_int8_feed_forward_workspace_bytes(count, 512, k, 1000, _lib.F32)
        assert both >= need - 4 * 4 * 512 * count + count * 4000
    # shares of K leave their sums: up to four of them, whole pieces of eight columns
    assert lib.dmoe_int8_linear_workspace_bytes(60, 4090, 11008, 1) == 4 * 60 * 4096 * 4
    assert lib.dmoe_int8_linear_workspace_bytes(0, 512, 128, 0) == 0 and lib.dmoe_int8_linear_workspace_bytes(1, 512, 65537, 0) == 0
    assert lib.dmoe_int8_linear_workspace_bytes(4, 0, 128, 0) == 0
    assert lib.dmoe_int8_feed_forward_workspace_bytes(4, 512, 128, 0, _lib.F32) == 0
    assert lib.dmoe_int8_feed_forward_workspace_bytes(4, 512, 128, 128, _lib.I32) == 0


# ------------------------------------------------------------------ the reference

def test_reference_rounding_is_the_types():
    g = np.random.default_rng(0)
    x = np.concatenate([g.standard_normal(4000) * 10.0 ** g.integers(-8, 4, 4000), ref.E4M3, -ref.E4M3])
    for dtype in ref.HALF:
        got = ref.through(x, dtype)
        assert (np.abs(got - x) <= ref.HALF[dtype] * np.abs(x) + ref.SMALL[dtype]).all()
        values = torch.from_numpy(got).to(dtype).double().numpy()
        assert np.array_equal(values, got)  # of the type
        assert np.array_equal(ref.through(got, dtype), got)


def test_reference_codes():
    assert np.array_equal(ref.E4M3, torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())
    y = np.random.default_rng(1).standard_normal((6, 256))
    y[5, 7] = np.inf
    codes, scales = ref.int8(y)
    assert np.isnan(scales[5]) and not codes[5].any() and (np.abs(codes).max(1)[:5] == 127).all()
    assert (np.abs(codes[:5] * scales[:5, None] - y[:5]) <= scales[:5, None] * 0.5 * (1 + 2.0 ** -20)).all()
    values, scales = ref.e4m3(y, 128)
    assert np.isnan(scales[5, 0]) and np.isfinite(scales[5, 1])
    x = np.random.default_rng(2).standard_normal((3, 64)).astype(np.float32)
    x[:, 0] = 448  # the scale is 1 up to its rounding: codes of a plain cast
    values, scales = ref.e4m3(x.astype(np.float64), 64)
    if (scales == 1).all():
        assert np.array_equal(values, torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy())


def test_reference_feed_forward_brackets_a_plain_one():
    g = np.random.default_rng(3)
    codes, scales = ref.int8(g.standard_normal((5, 64)))
    w, v = g.integers(-128, 128, (96, 64)).astype(float), g.integers(-128, 128, (20, 48)).astype(float)
    ws, vs = np.full(96, 0.002), np.full(20, 0.002)
    low, high = ref.feed_forward(codes, scales, w, ws, v, vs, BF16, "silu")
    first, _ = ref.product(codes, scales, w, ws)
    c, s = ref.int8(ref.through(ref.act(first[:, :48], "silu")[0] * first[:, 48:], BF16))
    out, _ = ref.product(c, s, v, vs)
    assert (low <= out).all() and (out <= high).all()


# ------------------------------------------------------------------ blocks

def test_dense_block_refusals():
    ffn = Int8FeedForward(i8(8, 32), torch.ones(8), i8(32, 4), torch.ones(32))
    with pytest.raises(ValueError, match="one width"):
        DenseBlock(RmsNorm(torch.ones(31), quant="int8"), ffn)
    with pytest.raises(ValueError, match="one width"):
        DenseBlock(RmsNorm(torch.ones(32)), Int8FeedForward(i8(8, 32), torch.ones(8), i8(33, 4), torch.ones(33)))
    with pytest.raises(ValueError, match="rows or 8-bit integers"):
        DenseBlock(RmsNorm(torch.ones(32), quant="fp8"), ffn)
    block = DenseBlock(RmsNorm(torch.ones(32), quant="int8"), ffn)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        block(torch.zeros(2, 32))


def test_attention_block_takes_rows_in_8_bits_for_8_bit_projections_only():
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device="cpu")
    batch = PagedBatch(torch.ones(2, 2).int(), torch.ones(2).int())
    x, residual = QuantRows(i8(2, 32), torch.ones(2)), torch.zeros(2, 32)
    linear = [torch.nn.Linear(32, 256), torch.nn.Linear(32, 128), torch.nn.Linear(32, 128), torch.nn.Linear(256, 32)]
    with torch.no_grad(), pytest.raises(ValueError, match="needs Int8Linear projections"):
        AttentionBlock(*linear, cache, heads=4)(x, residual, batch)
    with pytest.raises(ValueError, match="attn_input and residual"):
        AttentionBlock(*linear, cache, heads=4)(x, residual[:, :16], batch)
    eight = [Int8Linear.from_linear(m) for m in linear]
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        AttentionBlock(*eight, cache, heads=4)(x, residual, batch)


def test_a_capture_is_not_the_first_to_need_the_status_word(monkeypatch):
    device = torch.device("cuda", 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="once eagerly"):
        int8._status(device)
    assert device not in int8._STATES


def test_scales_that_need_gradients_are_refused():
    scales = torch.ones(2, requires_grad=True)
    for make in (QuantRows, Int8Weight):
        with pytest.raises(ValueError, match="scales needs gradients"):
            make(i8(2, 32), scales)
        with torch.no_grad():
            make(i8(2, 32), scales)
