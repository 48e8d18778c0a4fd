"""GPU: norms and rows in 8 bits, products of 8-bit integers and the gated
feed-forward block against 64-bit numpy statements of their definitions."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rows8_reference as ref
from conftest import print_case
from drama_moe import _lib
from drama_moe._lib import STATUS_NON_FINITE
from drama_moe.int8 import (Int8FeedForward, Int8Linear, Int8Weight, QuantRows, int8_feed_forward, int8_linear,
                            quantize_rows)
from drama_moe.norm import RmsNorm, rms_norm
from drama_moe.offload import device_state

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def status(device):
    word = device_state(device).status
    value = int(word.item())
    word.zero_()
    return value


def stream(rows, cols, dtype, g, size=1.0):
    x = torch.randn(rows, cols, generator=g) * (1 + 15 * (torch.rand(cols, generator=g) < 0.02)) * size
    return (x * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype)


def matrix(n, k, g):
    codes = (torch.randn(n, k, generator=g) * 40).round().clamp(-128, 127).to(torch.int8)
    return codes, torch.exp(0.3 * torch.randn(n, generator=g)) * (k ** -0.5 / 40)


def near(got, want, size, dtype):
    """|got - want| within the fp32 steps (six of 2^-24 of the magnitudes that meet) and half a step of the result."""
    got = ref.wide(got)
    slack = 6 * 2.0 ** -24 * size
    slack = slack + ref.HALF[dtype] * (np.abs(want) + slack) + ref.SMALL[dtype]
    off = np.abs(got - want) - slack
    assert got.shape == want.shape and not np.isnan(got).any() and off.max(initial=-1.0) <= 0, \
        f"off by {off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"


def same_rows8(q, values, scales):
    assert np.array_equal(ref.wide(q.scales).ravel(), scales.ravel(), equal_nan=True)
    got = q.values.float().cpu().double().numpy()
    assert np.array_equal(got, values), f"{(got != values).sum()} codes differ"
    rows, cols = q.shape
    width = -(-cols // 128) * 128
    if rows:  # the zeros behind the columns
        held = q.values.view(torch.int8).as_strided((rows, width), (q.values.stride(0), 1))
        assert not held[:, cols:].any()


def check_norm(cuda, rows, cols, dtype, quant, *, residual=True, keep=True, offset=0.0, weight_dtype=None, eps=1e-6, seed=0):
    print_case("norm", rows, cols, dtype, quant, residual, keep, offset)
    g = torch.Generator().manual_seed(seed + rows * 7 + cols)
    x, add = stream(rows, cols, dtype, g), stream(rows, cols, dtype, g, 2.0)
    weight = (0.2 * torch.randn(cols, generator=g) + 1 - offset).to(weight_dtype or dtype)
    made = rms_norm(x.to(cuda), weight.to(cuda), residual=add.to(cuda) if residual else None, eps=eps, offset=offset,
                    quant=quant, rows=keep)
    h, y = ref.norm(ref.wide(x), ref.wide(add) if residual else None, ref.wide(weight), dtype, eps=eps, offset=offset)
    assert np.array_equal(ref.wide(made.hidden), h)
    if keep:
        near(made.rows, y, np.abs(y), dtype)
    else:
        assert made.rows is None
    if quant == "int8":
        same_rows8(made.quant, *ref.int8(y))
    elif quant is not None:
        same_rows8(made.quant, *ref.e4m3(y, 128 if quant == "fp8-128" else cols))
    else:
        assert made.quant is None
    assert status(cuda) == 0


@pytest.mark.parametrize("cols", [1, 7, 8, 33, 128, 511, 513, 1000, 1025, 2048, 2501, 4096, 5000, 8192, 16000, 20001, 40000, 65536])
def test_norm_of_all_widths(cuda, cols):
    status(cuda)
    check_norm(cuda, 5, cols, torch.bfloat16, "int8")
    check_norm(cuda, 3, cols, torch.float16, "fp8", residual=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("quant", [None, "int8", "fp8", "fp8-128"])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_of_all_types(cuda, dtype, quant, residual):
    status(cuda)
    for rows, cols in ((1, 384), (257, 640), (66, 2048), (9, 11008)):
        check_norm(cuda, rows, cols, TYPES[dtype], quant, residual=residual, keep=quant is None or rows % 2 == 1)
    check_norm(cuda, 30, 1152, TYPES[dtype], quant, residual=residual, offset=1.0, weight_dtype=torch.float32)
    check_norm(cuda, 31, 1152, TYPES[dtype], quant, residual=residual, offset=1.0, weight_dtype=torch.bfloat16, eps=1e-2)


def test_norm_of_many_rows(cuda):
    """Codes of many values: every border that 32 bits could miss is one of them."""
    status(cuda)
    check_norm(cuda, 1500, 4096, torch.bfloat16, "int8")
    check_norm(cuda, 1500, 4096, torch.float32, "int8", residual=False)
    check_norm(cuda, 1500, 4096, torch.bfloat16, "fp8-128")
    check_norm(cuda, 1500, 4096, torch.float32, "fp8", residual=False)


def test_norm_where_rows_lie_apart(cuda):
    """Row strides of any size, columns of a wider tensor, one residual row for all, leading dimensions."""
    print_case("norm strides")
    g = torch.Generator().manual_seed(3)
    big = stream(40, 999, torch.float16, g).to(cuda)
    weight = (torch.rand(333, generator=g) + 0.5).half().to(cuda)
    for x in (big[:, 1:334], big[::3, 5:338], big[:, 600:933], big[3:4, 7:340]):
        add = big[:1, 2:335].expand(x.shape)
        a = rms_norm(x, weight, residual=add, quant="int8", rows=True)
        b = rms_norm(x.contiguous(), weight, residual=add.contiguous(), quant="int8", rows=True)
        for s, t in ((a.hidden, b.hidden), (a.rows, b.rows), (a.quant.values, b.quant.values), (a.quant.scales, b.quant.scales)):
            assert torch.equal(s, t)
        h, y = ref.norm(ref.wide(x), ref.wide(add), ref.wide(weight), torch.float16, eps=1e-6)
        same_rows8(a.quant, *ref.int8(y))
        assert np.array_equal(ref.wide(a.hidden), h)
    x = big[:, :333].reshape(2, 4, 5, 333)
    made = rms_norm(x, weight, residual=x, quant="int8", rows=True)
    assert made.hidden.shape == made.rows.shape == x.shape and made.quant.shape == (40, 333)
    flat = rms_norm(x.reshape(40, 333), weight, residual=x.reshape(40, 333), quant="int8", rows=True)
    assert torch.equal(made.rows.reshape(40, 333), flat.rows) and torch.equal(made.quant.values, flat.quant.values)
    x = big.t()[:333].t()  # columns apart: copied
    assert torch.equal(rms_norm(big.t().contiguous().t()[:, :333], weight).rows, rms_norm(x, weight).rows)
    none = rms_norm(big[:0, :333], weight, residual=big[:0, :333], quant="int8", rows=True)
    assert none.hidden.shape == none.rows.shape == none.quant.shape == (0, 333)


def test_norm_of_odd_values(cuda):
    """Zeros, tiny and huge rows; an infinity or NaN spoils its row (group) alone and is flagged."""
    print_case("norm odd values")
    status(cuda)
    weight = torch.ones(256)
    x = torch.randn(8, 256, generator=torch.Generator().manual_seed(1))
    x[0] = 0
    x[1] *= 1e-20
    x[2] *= 1e37
    x[3] *= 1e-42
    for quant in ("int8", "fp8", "fp8-128"):
        made = rms_norm(x.to(cuda), weight.to(cuda), quant=quant)
        _, y = ref.norm(ref.wide(x), None, ref.wide(weight), torch.float32, eps=1e-6)
        want = ref.int8(y) if quant == "int8" else ref.e4m3(y, 128 if quant == "fp8-128" else 256)
        same_rows8(made.quant, *want)
    assert status(cuda) == 0
    for bad in (float("inf"), float("-inf"), float("nan")):
        z = x.clone()
        z[5, 200] = bad
        for quant in ("int8", "fp8"):
            made = rms_norm(z.to(cuda), weight.to(cuda), quant=quant, rows=True)
            assert status(cuda) == STATUS_NON_FINITE
            assert torch.isnan(made.quant.scales).nonzero().flatten().tolist() == [5]
            assert not made.quant.values[5].float().any()
            assert torch.isnan(made.rows[5]).any() and not torch.isnan(made.rows[[0, 1, 2, 3, 4, 6, 7]]).any()
            assert torch.isnan(made.quant.dequantize(torch.float32)).nonzero()[:, 0].unique().tolist() == [5]
        made = rms_norm(z.to(cuda), weight.to(cuda), quant="fp8-128")
        assert status(cuda) == STATUS_NON_FINITE and torch.isnan(made.quant.scales[5, 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 127), (13, 8192), (64, 513), (300, 2501), (2, 16385), (1, 65536)])
def test_rows_to_integers(cuda, dtype, rows, cols):
    print_case("quantize", dtype, rows, cols)
    status(cuda)
    x = stream(rows, cols, TYPES[dtype], torch.Generator().manual_seed(rows + cols), 0.01)
    q = quantize_rows(x.to(cuda))
    codes, scales = ref.int8(ref.wide(x))
    same_rows8(q, codes, scales)
    for out in TYPES.values():
        assert np.array_equal(ref.wide(q.dequantize(out)),
                              ref.through((codes * scales[:, None]).astype(np.float32), out))
    assert status(cuda) == 0


def test_rows_on_borders(cuda):
    """Quotients that are exactly between two codes go to the even one, next to them to the nearer one."""
    print_case("quantize borders")
    for top in (127.0, 381.0, 127 * 2.0 ** -20, 127 * 2.0 ** -140 * 2.0 ** 100, 254.0):
        step = np.float32(top) * (np.float32(1) / np.float32(127))
        ties = (np.arange(-126, 127) + 0.5) * float(step)
        x = np.concatenate([[top], ties]).astype(np.float32)
        x = np.stack([x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf))])
        x[:, 0] = top
        q = quantize_rows(torch.from_numpy(x).to(cuda))
        same_rows8(q, *ref.int8(x.astype(np.float64)))
    v = ref.E4M3
    middle = (v[1:] + v[:-1]) / 2
    x = np.concatenate([[448.0], v, middle, -middle]).astype(np.float32)
    x = np.stack([x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf))])
    x[:, 0] = 448
    # a gain that undoes the norm's factor up to its rounding: the quotients lie on and around the borders
    y = x / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True))
    made = rms_norm(torch.from_numpy(x).to(cuda), torch.ones(x.shape[1], device=cuda), eps=0.0, quant="fp8")
    same_rows8(made.quant, *ref.e4m3(ref.norm(x.astype(np.float64), None, np.ones(x.shape[1]), torch.float32, eps=0.0)[1], x.shape[1]))
    assert y.shape == x.shape


def test_rows_that_are_not_finite(cuda):
    print_case("quantize not finite")
    status(cuda)
    w, ws = matrix(40, 300, torch.Generator().manual_seed(1))
    weight = Int8Weight(w.to(cuda), ws.to(cuda))
    for rows in (2, 3, 20, 70, 300):  # every way to a product
        x = torch.randn(rows, 300, generator=torch.Generator().manual_seed(rows))
        clean = int8_linear(x.to(cuda), weight)
        assert status(cuda) == 0
        x[1, 299] = float("nan")
        out = int8_linear(x.to(cuda), weight)
        assert status(cuda) == STATUS_NON_FINITE
        assert torch.isnan(out[1]).all()
        keep = [i for i in range(rows) if i != 1]
        assert torch.equal(out[keep], clean[keep])


def check_linear(cuda, rows, k, n, dtype, *, given=False, bias=False, residual=False, out=None):
    print_case("linear", rows, k, n, dtype, given, bias, residual, out)
    g = torch.Generator().manual_seed(rows * 31 + k * 7 + n)
    w, ws = matrix(n, k, g)
    x = stream(rows, k, dtype, g)
    b = torch.randn(n, generator=g) if bias else None
    out = out or dtype
    r = stream(rows, n, out, g) if residual else None
    codes, scales = ref.int8(ref.wide(x))
    weight = Int8Weight(w.to(cuda), ws.to(cuda))
    source = x.to(cuda)
    if given:
        source = QuantRows(torch.from_numpy(codes).to(torch.int8).to(cuda), torch.from_numpy(scales).float().to(cuda))
    got = int8_linear(source, weight, bias=b.to(cuda) if bias else None, residual=r.to(cuda) if residual else None, dtype=out)
    want, size = ref.product(codes, scales, ref.wide(w), ref.wide(ws), ref.wide(b) if bias else None,
                             ref.wide(r) if residual else None)
    near(got, want, size, out)
    return got


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 255, 257, 700])
def test_linear_of_all_row_counts(cuda, rows):
    check_linear(cuda, rows, 384, 200, torch.bfloat16)
    check_linear(cuda, rows, 200, 77, torch.float16, given=True, bias=True, residual=True)


@pytest.mark.parametrize("k", [1, 15, 16, 17, 64, 100, 127, 128, 129, 255, 1000, 2048, 4100, 16400])
def test_linear_of_all_depths(cuda, k):
    for rows in (1, 4, 20, 60, 130, 300):
        check_linear(cuda, rows, k, 48, torch.bfloat16, given=rows == 20, bias=True)


@pytest.mark.parametrize("n", [1, 3, 15, 16, 17, 31, 127, 129, 255, 257, 1000, 5003])
def test_linear_of_all_widths(cuda, n):
    for rows in (1, 18, 64, 200):
        check_linear(cuda, rows, 256, n, torch.float16, residual=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_linear_of_all_types(cuda, dtype, out):
    for rows in (2, 40, 150):
        check_linear(cuda, rows, 300, 100, TYPES[dtype], bias=True, residual=True, out=TYPES[out])


def test_linear_in_large_tiles(cuda):
    """Enough tiles to fill the chip, ragged at both ends and along K."""
    check_linear(cuda, 4000, 1000, 4500, torch.bfloat16, residual=True)
    check_linear(cuda, 4097, 130, 4097, torch.float16, given=True)
    check_linear(cuda, 1100, 2048, 4096, torch.bfloat16)
    check_linear(cuda, 1300, 300, 5000, torch.bfloat16, bias=True)


@pytest.mark.parametrize("rows", [1, 10, 40, 65, 300])
def test_linear_holds_the_largest_sums(cuda, rows):
    """2^16 products of -128 by -128, and by 127: the integers do not wrap."""
    print_case("linear largest", rows)
    k = 65536
    codes = torch.full((rows, k), -128, dtype=torch.int8)
    w = torch.full((3, k), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 127
    x = QuantRows(codes.to(cuda), torch.ones(rows, device=cuda))
    got = int8_linear(x, Int8Weight(w.to(cuda), torch.ones(3, device=cuda)), dtype=torch.float32).cpu()
    assert (got == torch.tensor([2.0 ** 30, -127 * 2.0 ** 23, 2.0 ** 22])).all()


@pytest.mark.parametrize("rows", [1, 3, 17, 130])
def test_linear_where_operands_lie_apart(cuda, rows):
    """Matrices and rows out of larger tensors, at any offset; leading dimensions."""
    print_case("linear strides", rows)
    g = torch.Generator().manual_seed(rows)
    held, ws = matrix(90, 400, g)
    held = held.to(cuda)
    x = stream(rows, 500, torch.bfloat16, g).to(cuda)
    add = stream(rows, 61, torch.bfloat16, g).to(cuda)
    for w, cols in ((held[20:70, :304], 304), (held[1::2, 3:300], 297), (held[:, 16:316], 300), (held[5:6, :256], 256)):
        scales = ws[:w.shape[0]].to(cuda)
        weight = Int8Weight(w, scales)
        plain = Int8Weight(w.clone(memory_format=torch.contiguous_format), scales.clone())
        rows_in = x[:, 11:11 + cols]
        n = w.shape[0]
        extra = add[:, 1:1 + n] if n <= 60 else None
        a = int8_linear(rows_in, weight, residual=extra)
        b = int8_linear(rows_in.contiguous(), plain, residual=extra.contiguous() if extra is not None else None)
        assert torch.equal(a, b)
        want, size = ref.product(*ref.int8(ref.wide(rows_in)), ref.wide(w), ref.wide(scales),
                                 residual=ref.wide(extra) if extra is not None else None)
        near(a, want, size, torch.bfloat16)
    weight = Int8Weight(held, ws.to(cuda))
    many = x[:, :400].reshape(1, rows, 1, 400)
    assert torch.equal(int8_linear(many, weight).reshape(rows, 90), int8_linear(x[:, :400], weight))
    assert int8_linear(x[:0, :400], weight).shape == (0, 90)
    one = int8_linear(x[0, :400], weight)  # a vector
    assert one.shape == (90,) and torch.equal(one, int8_linear(x[:1, :400], weight)[0])
    wide = x[:1, :400].expand(rows, 400)  # one row for all
    assert torch.equal(int8_linear(wide, weight), one.expand(rows, 90))


def test_a_row_does_not_depend_on_its_call(cuda):
    """The same row in calls of every size: the same bits."""
    print_case("linear across calls")
    g = torch.Generator().manual_seed(8)
    w, ws = matrix(500, 1100, g)
    weight = Int8Weight(w.to(cuda), ws.to(cuda))
    x = stream(3000, 1100, torch.bfloat16, g).to(cuda)
    whole = int8_linear(x, weight, dtype=torch.float32)
    for at, rows in ((0, 1), (7, 3), (100, 5), (64, 30), (1, 64), (900, 65), (2000, 400)):
        assert torch.equal(int8_linear(x[at:at + rows], weight, dtype=torch.float32), whole[at:at + rows])


def check_ffn(cuda, rows, k, inter, n, dtype, act="silu", *, given=False, residual=True, seed=0):
    print_case("ffn", rows, k, inter, n, dtype, act, given, residual)
    g = torch.Generator().manual_seed(seed + rows * 31 + k * 7 + inter)
    w, ws = matrix(2 * inter, k, g)
    v, vs = matrix(n, inter, g)
    x = stream(rows, k, dtype, g, 0.4)
    r = stream(rows, n, dtype, g) if residual else None
    codes, scales = ref.int8(ref.wide(x))
    source = x.to(cuda)
    if given:
        source = QuantRows(torch.from_numpy(codes).to(torch.int8).to(cuda), torch.from_numpy(scales).float().to(cuda))
    got = int8_feed_forward(source, Int8Weight(w.to(cuda), ws.to(cuda)), Int8Weight(v.to(cuda), vs.to(cuda)), activation=act,
                            residual=r.to(cuda) if residual else None, dtype=dtype)
    low, high = ref.feed_forward(codes, scales, ref.wide(w), ref.wide(ws), ref.wide(v), ref.wide(vs), dtype, act,
                                 ref.wide(r) if residual else None)
    out = ref.wide(got)
    slack = ref.HALF[dtype] * np.maximum(np.abs(low), np.abs(high)) + ref.SMALL[dtype]
    assert (out >= low - slack).all() and (out <= high + slack).all(), \
        f"{np.maximum(low - slack - out, out - high - slack).max()} outside the bounds"
    # the bounds say something: next to the results they are narrow
    assert (high - low).mean() < 0.2 * np.sqrt((out * out).mean())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_feed_forward_of_all_row_counts(cuda, dtype, act):
    for rows in (1, 2, 4, 5, 17, 40, 65, 200):
        check_ffn(cuda, rows, 256, 272, 192, TYPES[dtype], act, given=rows == 5, residual=rows % 2 == 0)


@pytest.mark.parametrize("k,inter,n", [(1, 1, 1), (17, 15, 3), (130, 129, 131), (1000, 65, 257), (64, 1000, 100), (2048, 768, 2048)])
def test_feed_forward_of_all_sizes(cuda, k, inter, n):
    for rows in (1, 3, 20, 70, 150):
        check_ffn(cuda, rows, k, inter, n, torch.bfloat16)


def test_feed_forward_in_large_tiles(cuda):
    check_ffn(cuda, 2100, 500, 2200, 600, torch.bfloat16)


@pytest.mark.parametrize("rows", [1, 20, 100])
def test_activation_over_its_whole_range(cuda, rows):
    """Gates from far below zero to far above; a matrix that gives the hidden rows back shows each by itself."""
    print_case("ffn activation", rows)
    inter = 120
    gates = np.concatenate([np.linspace(-127, 127, inter - 20), np.linspace(-1, 1, 20)])
    w = torch.zeros(2 * inter, 16, dtype=torch.int8)
    w[:inter, 0] = torch.from_numpy(np.rint(gates)).to(torch.int8)
    w[inter:, 1] = 100
    v = 127 * torch.eye(inter).to(torch.int8)
    one = torch.ones(2 * inter) * 0.1
    x = torch.zeros(rows, 16)
    x[:, 0], x[:, 1] = 127.0, 127.0
    back = torch.full((inter,), 1 / 127)
    for act in ("silu", "gelu_tanh"):
        got = ref.wide(int8_feed_forward(x.to(cuda), Int8Weight(w.to(cuda), one.to(cuda)), Int8Weight(v.to(cuda), back.to(cuda)),
                                         activation=act, dtype=torch.float32))
        z = 127 * np.rint(gates) * np.float64(np.float32(0.1))
        want = ref.act(z, act)[0] * (127 * 100 * np.float64(np.float32(0.1)))
        step = np.abs(want).max() / 127
        assert np.abs(got - want).max() <= step * 0.5001 + 1e-6 * np.abs(want).max()


def test_modules(cuda):
    """Int8Linear and Int8FeedForward are the functions on their matrices, also after they moved; odd columns too."""
    print_case("modules")
    torch.manual_seed(4)
    linear = torch.nn.Linear(100, 36)
    q = Int8Linear.from_linear(linear, device=cuda)
    x = torch.randn(7, 100).to(cuda)
    exact = ref.wide(x) @ ref.wide(linear.weight).T + ref.wide(linear.bias)
    got = ref.wide(q(x))
    # half a step of each row of x and of the matrix, against the other's magnitudes
    sx, sw = ref.wide(x.abs().amax(1)) / 254, ref.wide(linear.weight.abs().amax(1)) / 254
    bound = sx[:, None] * np.abs(ref.wide(linear.weight)).sum(1) + np.abs(ref.wide(x)).sum(1)[:, None] * sw + 100 * sx[:, None] * sw
    assert (np.abs(got - exact) <= bound * 1.001).all()
    moved = Int8Linear.from_linear(linear).to(cuda)
    assert torch.equal(moved(x), q(x))
    other = Int8Linear.from_linear(torch.nn.Linear(100, 36), device=cuda)
    other.load_state_dict(q.state_dict())
    assert torch.equal(other(x), q(x))
    assert torch.equal(q(quantize_rows(x), dtype=torch.float32), q(x))
    gate, up, down = (torch.nn.Linear(a, b, bias=False) for a, b in ((50, 70), (50, 70), (70, 50)))
    block = Int8FeedForward.from_linears(gate, up, down, device=cuda)
    y = torch.randn(5, 50).to(cuda)
    w, v = block.gate_up, block.down
    assert torch.equal(block(y, residual=y),
                       int8_feed_forward(y, Int8Weight(w.qweight[:, :50], w.scales), Int8Weight(v.qweight[:, :70], v.scales), residual=y))
    norm = RmsNorm(torch.rand(50).to(cuda), quant="int8")
    made = norm(y, y)
    assert torch.equal(made.hidden, y + y) and made.rows is None
    assert torch.equal(block(made.quant, residual=made.hidden), block(made.quant, residual=made.hidden))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_over_the_whole_range(cuda, dtype):
    """Rows from the smallest to the largest numbers, whose squares and whose norms' factors pass 32 bits."""
    print_case("norm range", dtype)
    status(cuda)
    g = torch.Generator().manual_seed(11)
    sizes = (1e-44, 1e-39, 1e-37, 1e-30, 1e-25, 1e-10, 1.0, 1e15, 1e20, 1e30, 1e37)
    x = torch.randn(len(sizes), 640, generator=g).clamp(-4, 4) * torch.tensor(sizes)[:, None]
    x[0, 0] = x[1, 0] = 1e-38  # bf16 has no 1e-44
    x = x.to(TYPES[dtype])
    for gain in (1.0, 1e-6, 3.0):
        weight = (torch.rand(640, generator=g) + 0.5) * gain
        for eps in (0.0, 1e-60, 1e-6):
            h, y = ref.norm(ref.wide(x), None, ref.wide(weight), TYPES[dtype], eps=eps)
            for quant in ("int8", "fp8", "fp8-128"):
                print_case("norm range", dtype, gain, eps, quant)
                made = rms_norm(x.to(cuda), weight.to(cuda), eps=eps, quant=quant, rows=True)
                near(made.rows, y, np.abs(y), TYPES[dtype])
                same_rows8(made.quant, *(ref.int8(y) if quant == "int8" else ref.e4m3(y, 128 if quant == "fp8-128" else 640)))
    assert status(cuda) == 0


@pytest.mark.parametrize("cols", [8, 333, 1000, 2501, 9001])
def test_outputs_in_their_inputs_places(cuda, cols):
    """hidden in x's or residual's memory, a product's result in its residual's."""
    print_case("in place", cols)
    g = torch.Generator().manual_seed(cols)
    lib, stream_of = _lib.library(), torch.cuda.current_stream(cuda).cuda_stream
    desc = lambda t: _lib.Rows(t.data_ptr(), t.stride(0), _lib.dtype_code(t.dtype))  # noqa: E731
    for dtype in TYPES.values():
        for rows in (3, 700):
            x, add = stream(rows, cols, dtype, g).to(cuda), stream(rows, cols, dtype, g).to(cuda)
            weight = (torch.rand(cols, generator=g) + 0.5).to(cuda)
            want = rms_norm(x, weight, residual=add)
            for place in (0, 1):
                both = [x.clone(), add.clone()]
                out = torch.empty_like(x)
                _lib.check(lib.dmoe_rms_norm(desc(both[0]), desc(both[1]), rows, cols, weight.data_ptr(), _lib.F32, 0.0, 1e-6,
                                             desc(both[place]), desc(out), None, None, stream_of))
                assert torch.equal(both[place], want.hidden) and torch.equal(out, want.rows)
                assert torch.equal(both[1 - place], (x, add)[1 - place])
    codes, scales = matrix(cols, 90, g)
    weight = Int8Weight(codes.to(cuda), scales.to(cuda))
    for rows in (2, 20, 70, 700):
        x, add = quantize_rows(stream(rows, 90, torch.bfloat16, g).to(cuda)), stream(rows, cols, torch.bfloat16, g).to(cuda)
        want = int8_linear(x, weight, residual=add)
        need = lib.dmoe_int8_linear_workspace_bytes(rows, cols, 90, 1)
        room = torch.empty(need + 256, dtype=torch.uint8, device=cuda)
        _lib.check(lib.dmoe_int8_linear(None, x.desc, rows, weight.desc, None, desc(add), desc(add), room.data_ptr(), need, None,
                                        stream_of))
        assert torch.equal(add, want)


def test_offsets_beyond_32_bits(cuda):
    """Rows, matrices, results and 8-bit rows of over 4 GiB: their ends are those of calls on the ends alone."""
    print_case("linear with a matrix over 4 GiB")
    n, k = 66000, 65536
    codes = torch.randint(-128, 128, (n, k), dtype=torch.int8, device=cuda)
    scales = torch.rand(n, device=cuda)
    whole, end = Int8Weight(codes, scales), Int8Weight(codes[-300:], scales[-300:])
    for rows in (1, 40, 70, 300):
        x = torch.randn(rows, k, device=cuda)
        assert torch.equal(int8_linear(x, whole)[:, -300:], int8_linear(x, end))
    print_case("linear with rows over 4 GiB")
    rows = codes[:, :k]  # in 8 bits
    few = Int8Weight(codes[:130].clone(), scales[:130])
    q = QuantRows(rows, scales)
    assert q.values.data_ptr() == codes.data_ptr()
    assert torch.equal(int8_linear(q, few)[-100:], int8_linear(QuantRows(rows[-100:], scales[-100:]), few))
    assert torch.equal(q.dequantize(torch.float16)[-3:], QuantRows(rows[-3:], scales[-3:]).dequantize(torch.float16))
    del codes, whole, end, rows, q
    print_case("gate and up of almost 2 GiB apart")
    held = torch.randint(-128, 128, (2 * 20000, 50000), dtype=torch.int8, device=cuda)
    near_by = held[:, 1600:1700].contiguous()
    down = Int8Weight(held[:50, :20000].contiguous(), scales[:50])
    for rows in (1, 40, 100, 1100):
        x = torch.randn(rows, 100, device=cuda) * 0.01
        a = int8_feed_forward(x, Int8Weight(held[:, 1600:1700], scales[:40000] * 1e-3), down)
        assert torch.equal(a, int8_feed_forward(x, Int8Weight(near_by, scales[:40000] * 1e-3), down)) and torch.isfinite(a).all()
    del held, near_by, down
    print_case("norm of rows over 4 GiB")
    x = torch.randn(70000, 40000, device=cuda).bfloat16()
    weight = torch.rand(40000, device=cuda)
    made, alone = (rms_norm(t, weight, residual=t, quant="int8", rows=True) for t in (x, x[-9:]))
    for a, b in ((made.hidden, alone.hidden), (made.rows, alone.rows), (made.quant.values, alone.quant.values),
                 (made.quant.scales, alone.quant.scales)):
        assert torch.equal(a[-9:], b)
    del x, made, alone
    print_case("results over 4 GiB")
    q, w = (torch.randint(-128, 128, (n, 128), dtype=torch.int8, device=cuda) for n in (70000, 32000))
    w = Int8Weight(w, scales[:32000])
    ones = torch.rand(70000, device=cuda)
    out = int8_linear(QuantRows(q, ones), w)
    assert torch.equal(out[-300:], int8_linear(QuantRows(q[-300:], ones[-300:]), w))
    del out
    torch.cuda.empty_cache()


def test_more_rows_than_a_launch_holds(cuda):
    print_case("rows of several launches")
    rows, tail = (1 << 21) + 5, (1 << 21) - 700
    weight = torch.rand(128, device=cuda)
    x, add = (torch.randn(rows, 128, device=cuda).half() for _ in range(2))
    for quant in ("int8", "fp8-128"):
        made, end = (rms_norm(x[at:], weight, residual=add[at:], quant=quant, rows=True) for at in (0, tail))
        for a, b in ((made.hidden, end.hidden), (made.rows, end.rows), (made.quant.values.view(torch.int8), end.quant.values.view(torch.int8)),
                     (made.quant.scales, end.quant.scales)):
            assert torch.equal(a[tail:], b)
        assert torch.equal(made.hidden[:tail], x[:tail] + add[:tail])
    del made, end, x, add
    print_case("the most rows of several waves each")
    one = torch.randn(1, 1100, device=cuda).bfloat16()
    q = quantize_rows(one.expand(1 << 24, 1100))
    first = quantize_rows(one)
    assert (q.scales == first.scales).all()
    for part in q.values.split(1 << 21):
        assert (part == first.values).all()
    out, same = q.dequantize(), first.dequantize()
    for part in out.split(1 << 21):
        assert (part == same).all()
    del q, out, part
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_with_bias_and_residual_does_not_depend_on_its_call(cuda, dtype):
    """The steps behind a sum are the same in every kernel, whatever surrounds the row."""
    print_case("rows with bias and residual across calls", dtype)
    g = torch.Generator().manual_seed(21)
    for k, n in ((1100, 500), (9000, 700), (4096, 4096)):
        w, ws = matrix(n, k, g)
        weight, bias = Int8Weight(w.to(cuda), ws.to(cuda)), torch.randn(n, generator=g).to(cuda)
        x, add = stream(3000, k, TYPES[dtype], g).to(cuda), stream(3000, n, TYPES[dtype], g).to(cuda)
        for b, r in ((bias, add), (bias, None), (None, add)):
            whole = int8_linear(x, weight, bias=b, residual=r)
            for at, rows in ((0, 1), (7, 3), (100, 5), (64, 30), (1, 64), (900, 65), (2000, 400), (100, 1100)):
                got = int8_linear(x[at:at + rows], weight, bias=b, residual=r[at:at + rows] if r is not None else None)
                assert torch.equal(got, whole[at:at + rows]), (k, n, rows, b is None, r is None)
    for k, inter, n in ((500, 700, 300), (2048, 1500, 2048), (4096, 6000, 128)):
        w, ws = matrix(2 * inter, k, g)
        v, vs = matrix(n, inter, g)
        up, down = Int8Weight(w.to(cuda), ws.to(cuda)), Int8Weight(v.to(cuda), vs.to(cuda))
        x, add = stream(3000, k, TYPES[dtype], g, 0.4).to(cuda), stream(3000, n, TYPES[dtype], g).to(cuda)
        for act in ("silu", "gelu_tanh"):
            whole = int8_feed_forward(x, up, down, activation=act, residual=add)
            for at, rows in ((0, 1), (7, 3), (100, 5), (64, 30), (1, 64), (900, 65), (2000, 400), (100, 1100)):
                got = int8_feed_forward(x[at:at + rows], up, down, activation=act, residual=add[at:at + rows])
                assert torch.equal(got, whole[at:at + rows]), (k, inter, n, act, rows)


def test_a_norms_row_does_not_depend_on_its_call(cuda):
    """Rows in calls of every size, held by other numbers of threads: the same bits.  (64-bit sums in another order move
    the root by 2^-52, over a border of 24 bits in one row of 2^27.)"""
    print_case("norm across calls")
    g = torch.Generator().manual_seed(31)
    for cols in (384, 1024, 2048, 2501, 5120, 8192, 11008, 14336):
        x, add = (stream(1500, cols, torch.bfloat16, g).to(cuda) for _ in range(2))
        weight = (torch.rand(cols, generator=g) + 0.5).to(cuda)
        for quant in ("int8", "fp8", "fp8-128" if cols % 128 == 0 else "int8"):
            whole = rms_norm(x, weight, residual=add, quant=quant, rows=True)
            for at, rows in ((0, 1), (17, 30), (400, 256), (600, 257), (300, 1100)):
                got = rms_norm(x[at:at + rows], weight, residual=add[at:at + rows], quant=quant, rows=True)
                for a, b in ((got.hidden, whole.hidden), (got.rows, whole.rows), (got.quant.scales, whole.quant.scales),
                             (got.quant.values.view(torch.int8), whole.quant.values.view(torch.int8))):
                    assert torch.equal(a, b[at:at + rows]), (cols, quant, rows)
