"""GPU: products of 8-bit integers whose scales lie far apart, against their
64-bit statement, in every kernel that a product can take."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rows8_reference as ref
from conftest import print_case
from drama_moe.int8 import Int8Weight, QuantRows, int8_feed_forward, int8_linear

pytestmark = pytest.mark.gpu


def integers(rows, cols, g):
    return torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int8)


@pytest.mark.parametrize("rows", [1, 4, 20, 64, 70, 130, 300, 1100])
@pytest.mark.parametrize("channel", [1e36, 3e30, 2.0, 1.0, 1e-3, 1e-30, 1e-36, 1e-43])
def test_scales_far_apart(cuda, rows, channel):
    """Results of ordinary size from scales near both ends of fp32: no step on the way leaves its range."""
    print_case("int8 scales far apart", rows, channel)
    g = torch.Generator().manual_seed(rows)
    for k, n in ((300, 90), (6000, 90)):
        codes, w = integers(rows, k, g), integers(n, k, g)
        ws = (torch.rand(n, generator=g) + 0.5) * channel
        size = min(1e-6 / channel, 1e37)
        xs = (torch.rand(rows, generator=g) + 0.5) * size
        ws[::3] *= -1
        for bias in (None, torch.randn(n, generator=g)):
            got = int8_linear(QuantRows(codes.to(cuda), xs.to(cuda)), Int8Weight(w.to(cuda), ws.to(cuda)),
                              bias=bias.to(cuda) if bias is not None else None, dtype=torch.float32)
            want, magnitude = ref.product(codes.double().numpy(), ref.wide(xs), w.double().numpy(), ref.wide(ws),
                                          ref.wide(bias) if bias is not None else None)
            # three roundings and the bias' of 2^-24 each, and half of the smallest step where a result lies below 2^-126
            assert np.isfinite(ref.wide(got)).all()
            assert (np.abs(ref.wide(got) - want) <= 4 * 2.0 ** -24 * magnitude + 2.0 ** -149).all()


@pytest.mark.parametrize("rows", [1, 20, 70, 300])
def test_gates_of_scales_far_apart(cuda, rows):
    """The same for the feed-forward block's first product: a matrix that gives the hidden rows back shows each."""
    print_case("int8 gate scales far apart", rows)
    g = torch.Generator().manual_seed(rows)
    k, inter = 200, 60
    codes, w = integers(rows, k, g), integers(2 * inter, k, g)
    plain, far = torch.rand(2 * inter, generator=g) * 1e-3 + 1e-3, 2.0 ** 125
    xs = torch.rand(rows, generator=g) + 1
    down = Int8Weight(127 * torch.eye(inter).to(torch.int8).to(cuda), torch.full((inter,), 1 / 127).to(cuda))
    a, b = (int8_feed_forward(QuantRows(codes.to(cuda), (xs / by).to(cuda)), Int8Weight(w.to(cuda), (plain * by).to(cuda)), down,
                              dtype=torch.float32) for by in (1.0, far))
    # powers of two: the same significands, so a and b differ by what the order of the two scales does to a last bit of gate
    # and up, (|y| + 1) 2^-22 of a hidden value; a code moves by one step at most
    assert torch.isfinite(b).all()
    step = a.abs().amax(1, keepdim=True) / 127
    assert ((a - b).abs() <= step * 1.001).all() and ((a - b).abs() > step * 0.5).float().mean() < 0.01
