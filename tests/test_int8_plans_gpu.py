"""GPU: every kernel that a product of 8-bit integers can take, gated ones too,
against the 64-bit statement; a row's bits across all of them; codes at and
next to the borders between E4M3 numbers."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rows8_reference as ref
from conftest import print_case
from drama_moe.int8 import Int8FeedForward, Int8Weight, QuantRows, int8_feed_forward, int8_linear, quantize_rows
from drama_moe.norm import RmsNorm, rms_norm
from int8_plan_cases import GATED, PRODUCTS, T64, T128, WAVES
from test_rows8_gpu import check_linear, matrix, same_rows8, stream

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.mark.parametrize("case", PRODUCTS, ids=lambda c: "-".join(map(str, c)))
def test_products_in_every_kernel(cuda, case):
    rows, k, n, _, _ = case
    check_linear(cuda, rows, k, n, torch.bfloat16)
    check_linear(cuda, rows, k, n, torch.float16, given=True, bias=True, residual=True)
    check_linear(cuda, rows, k, n, torch.float32, residual=True)


@pytest.mark.parametrize("case", WAVES, ids=lambda c: "-".join(map(str, c)))
def test_few_rows_in_workgroups_of_each_size(cuda, case):
    rows, k, n = case
    check_linear(cuda, rows, k, n, torch.bfloat16, given=True, bias=True)
    check_linear(cuda, rows, k, n, torch.float16, residual=True)


def check_gated(cuda, rows, k, inter, n, dtype, act, *, given, residual):
    """Within the interval that the fp32 steps of the hidden rows allow.  It widens with sqrt(inter) against the results (a
    row's scale by a step of the type), so what it tells apart is asked of it directly: a neighbour's results lie outside."""
    print_case("gated", rows, k, inter, n, dtype, act, given, residual)
    g = torch.Generator().manual_seed(rows * 31 + k * 7 + inter)
    (w, ws), (v, vs) = matrix(2 * inter, k, g), matrix(n, inter, g)
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
    outside = lambda t: (t < low - slack) | (t > high + slack)  # noqa: E731
    assert np.isfinite(out).all() and not outside(out).any()
    for axis in (0, 1):
        if out.shape[axis] > 1:
            assert outside(np.roll(out, 1, axis)).mean() > 0.5


@pytest.mark.parametrize("case", GATED, ids=lambda c: "-".join(map(str, c)))
def test_feed_forward_in_every_kernel(cuda, case):
    rows, k, inter, n, _, _ = case
    check_gated(cuda, rows, k, inter, n, torch.bfloat16, "silu", given=False, residual=True)
    check_gated(cuda, rows, k, inter, n, torch.float16, "gelu_tanh", given=True, residual=False)
    check_gated(cuda, rows, k, inter, n, torch.float32, "silu", given=True, residual=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("case", [c for c in GATED if c[-1] > 1 or c[-2] == T128], ids=lambda c: "-".join(map(str, c)))
def test_a_gated_row_does_not_depend_on_its_call(cuda, case, act, dtype):
    rows, k, inter, n, shape, _ = case
    print_case("gated rows across calls", case, act, dtype)
    g = torch.Generator().manual_seed(k)
    (w, ws), (v, vs) = matrix(2 * inter, k, g), matrix(n, inter, g)
    up, down = Int8Weight(w.to(cuda), ws.to(cuda)), Int8Weight(v.to(cuda), vs.to(cuda))
    x, add = stream(rows, k, TYPES[dtype], g, 0.4).to(cuda), stream(rows, n, TYPES[dtype], g).to(cuda)
    whole = int8_feed_forward(x, up, down, activation=act, residual=add)
    for at, part in ((0, 1), (5, 3), (2, 17), (1, 33)) + (((3, 64), (100, 65), (400, 700)) if shape != T64 else ()):
        got = int8_feed_forward(x[at:at + part], up, down, activation=act, residual=add[at:at + part])
        assert torch.equal(got, whole[at:at + part]), part


@pytest.mark.parametrize("dtype", TYPES)
def test_a_products_row_does_not_depend_on_its_kernel(cuda, dtype):
    """The same rows in calls that take the kernels in turn."""
    print_case("rows across kernels", dtype)
    g = torch.Generator().manual_seed(5)
    for k, n in ((130, 4480), (10200, 320)):
        (w, ws), bias = matrix(n, k, g), torch.randn(n, generator=g).to(cuda)
        weight = Int8Weight(w.to(cuda), ws.to(cuda))
        x, add = stream(4000, k, TYPES[dtype], g).to(cuda), stream(4000, n, TYPES[dtype], g).to(cuda)
        whole = int8_linear(x, weight, bias=bias, residual=add)
        for rows in (1, 20, 65, 100, 190, 600, 1100, 2048):
            assert torch.equal(int8_linear(x[:rows], weight, bias=bias, residual=add[:rows]), whole[:rows]), (k, rows)


@pytest.mark.parametrize("quant", ["fp8", "fp8-128"])
@pytest.mark.parametrize("scale", [1.0, 0.5, 2.0 ** 20])
def test_e4m3_codes_on_borders(cuda, quant, scale):
    """Rows of ones with eps 0 have the factor 1, and 448 fl32(1/448) is 1: the gains are the quotients.  All numbers, all
    middles between two and their neighbours in fp32."""
    print_case("e4m3 borders", quant, scale)
    v = ref.E4M3
    middle = (v[1:] + v[:-1]) / 2
    points = np.concatenate([v, middle, -v, -middle]).astype(np.float32)
    around = np.concatenate([points, np.nextafter(points, np.float32(np.inf)), np.nextafter(points, np.float32(-np.inf))])
    around = np.clip(around, -448, 448).astype(np.float32)
    groups = -(-len(around) // 127)  # the largest number first in each group
    gain = np.zeros((groups, 128), np.float32)
    gain[:, 0] = 448
    gain[:, 1:].flat[:len(around)] = around
    gain = gain.reshape(-1) * np.float32(scale)
    x = torch.ones(3, gain.size)
    made = rms_norm(x.to(cuda), torch.from_numpy(gain).to(cuda), eps=0.0, quant=quant)
    _, y = ref.norm(x.double().numpy(), None, gain.astype(np.float64), torch.float32, eps=0.0)
    assert np.array_equal(y, np.broadcast_to(gain, y.shape))
    values, scales = ref.e4m3(y, 128 if quant == "fp8-128" else gain.size)
    assert (scales == scale).all()  # the test's own claim: quotients are exactly the points
    ties = np.isin(np.abs(gain / np.float32(scale)), middle.astype(np.float32)).sum()
    assert ties >= 2 * len(middle)
    same_rows8(made.quant, values, scales)


def test_e4m3_codes_next_to_borders_of_other_scales(cuda):
    """Scales that are no powers of two: quotients near the middles, where 32 bits alone would miss the side."""
    print_case("e4m3 near borders")
    v = ref.E4M3
    middle = (v[1:] + v[:-1]) / 2
    for top in (1.0, 3.3, 1000.7, 1e-3):
        scale = np.float32(top) * np.float32(1 / 448)
        near = (middle * np.float64(scale)).astype(np.float32)
        x = np.concatenate([[top], near, np.nextafter(near, np.float32(np.inf)), np.nextafter(near, np.float32(0))]).astype(np.float32)
        x = x[np.abs(x) <= np.float32(top)]
        x[0] = top
        gain = torch.from_numpy(x)
        made = rms_norm(torch.ones(2, x.size, device=cuda), gain.to(cuda), eps=0.0, quant="fp8")
        y = np.broadcast_to(x.astype(np.float64), (2, x.size))
        same_rows8(made.quant, *ref.e4m3(y, x.size))


def test_a_modules_type_is_what_rows_in_8_bits_give(cuda):
    """QuantRows without a residual come out in the module's type, with one in the residual's."""
    print_case("module types")
    torch.manual_seed(4)
    for dtype in TYPES.values():
        gate, up, down = (torch.nn.Linear(a, b, bias=False) for a, b in ((50, 70), (50, 70), (70, 50)))
        block = Int8FeedForward.from_linears(gate, up, down, device=cuda, dtype=dtype)
        y = torch.randn(5, 50).to(cuda)
        made = RmsNorm(torch.rand(50).to(cuda), quant="int8")(y, y)
        w, v = block.gate_up._weight(), block.down._weight()
        out = block(made.quant)
        assert out.dtype is dtype and torch.equal(out, int8_feed_forward(made.quant, w, v, dtype=dtype))
        with_add = block(made.quant, residual=made.hidden)
        assert with_add.dtype is torch.float32
        assert torch.equal(with_add, int8_feed_forward(made.quant, w, v, residual=made.hidden, dtype=torch.float32))
        rows = quantize_rows(y)
        assert torch.equal(block.gate_up(rows), int8_linear(rows, w, dtype=dtype))
