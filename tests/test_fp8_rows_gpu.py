"""GPU: rows in E4M3, as a norm leaves them, through the FP8 experts."""
from __future__ import annotations

import pytest
import torch

from conftest import print_case
from drama_moe import fp8_decode, fp8_moe
from drama_moe.formats import FP8_DTYPE, StagedExperts, random_fp8_bank
from drama_moe.norm import rms_norm
from drama_moe.offload import HipExpertBackend

pytestmark = pytest.mark.gpu

HIDDEN, EXPERTS = 512, 12


def bank(cuda, layout="block", seed=3):
    made = random_fp8_bank(EXPERTS, HIDDEN, 256, layout=layout, generator=torch.Generator().manual_seed(seed))
    return StagedExperts(*(t.to(cuda) for t in made.buffers().values()))


def codes(rows, g, cuda):
    """E4M3 numbers of all sizes, none of them NaN."""
    return (torch.randn(rows, HIDDEN, generator=g) * 40).to(FP8_DTYPE).to(cuda)


def routes(pairs, g, cuda):
    return torch.randint(0, EXPERTS, (pairs,), generator=g).to(cuda), torch.rand(pairs, generator=g).to(cuda)


def spread(q, scales, ids, weights, staged):
    """How far two right results of a pair may be apart: gate and up [I] by a step of bf16 and by the fp32 steps of 512
    products (2^-18 of their magnitudes' sum), |silu'| <= 1.1, a hidden value by half a step of E4M3 in each result, 2^-4 of
    it or, of a subnormal, 2^-10 of the scale, the group's largest value by 448."""
    full = lambda w, s: w.double() * s.double().repeat_interleave(w.shape[0] // s.shape[0], 0) \
        .repeat_interleave(w.shape[1] // s.shape[1], 1)  # noqa: E731
    x = (q.double() * scales.double()[:, None]).expand(ids.numel(), HIDDEN)
    out = torch.zeros(ids.numel(), HIDDEN, dtype=torch.float64, device=q.device)
    for e in range(EXPERTS):
        at = (ids == e).nonzero().flatten()
        w13 = full(staged.w13_weight[e], staged.w13_scale_inv[e])
        w2 = full(staged.w2_weight[e], staged.w2_scale_inv[e])
        (g, u), (sg, su) = (x[at] @ w13.T).chunk(2, 1), (x[at].abs() @ w13.T.abs()).chunk(2, 1)
        dg, du = g.abs() * 2.0 ** -8 + sg * 2.0 ** -18, u.abs() * 2.0 ** -8 + su * 2.0 ** -18
        h = (g.abs() + dg) * (u.abs() + du)
        dh = 1.1 * dg * (u.abs() + du) + (g.abs() + dg) * du
        dh = dh + 2 * (h * 2.0 ** -4 + h.amax(1, keepdim=True) / 448 * 2.0 ** -10)
        out[at] = dh @ w2.T.abs() * weights[at].double()[:, None]
    return out


@pytest.mark.parametrize("layout", ["block", "channel"])
@pytest.mark.parametrize("pairs", [1, 7, 30, 200, 300, 2000])
def test_a_scale_a_row_is_that_scale_for_each_group(cuda, pairs, layout):
    """The same bits: with powers of two for the rows' scales no order of theirs matters.  Above 256 pairs a matrix's
    scales for each channel, no powers of two, are applied to a whole sum where the rows have one scale, and to the sums of
    128 columns where they have groups: fl(fl(a w) + fl(b w)) is not fl((a + b) w)."""
    print_case("experts on a scale a row", pairs, layout)
    g = torch.Generator().manual_seed(pairs)
    staged = bank(cuda, layout)
    for rows in {1, pairs}:
        q = codes(rows, g, cuda)
        scales = torch.exp2(torch.randint(-9, -3, (rows,), generator=g).float()).to(cuda)
        ids, weights = routes(pairs, g, cuda)
        each = fp8_decode.quantized_pairs(fp8_moe, q, scales[:, None].repeat(1, HIDDEN // 128), ids, weights, staged)
        assert torch.isfinite(each).all() and each.abs().max() > 0
        for given in (scales, scales[:, None], scales.repeat_interleave(3)[::3]):
            got = fp8_decode.quantized_pairs(fp8_moe, q, given, ids, weights, staged)
            if pairs > 256 and layout == "channel":
                assert ((got - each).abs() <= spread(q, scales, ids, weights, staged)).all()
            else:
                assert torch.equal(got, each)


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
def test_a_norms_rows_with_a_scale_each_reach_the_experts(cuda, rows):
    """What the experts make of the norm's E4M3 rows is what they make of the values those rows stand for."""
    print_case("norm with a scale a row before experts", rows)
    g = torch.Generator().manual_seed(rows)
    staged = bank(cuda)
    x = torch.randn(rows, HIDDEN, generator=g).bfloat16().to(cuda)
    weight = (torch.rand(HIDDEN, generator=g) + 0.5).bfloat16().to(cuda)
    made = rms_norm(x, weight, residual=x, quant="fp8").quant
    ids, weights = routes(rows, g, cuda)
    got = fp8_decode.quantized_pairs(fp8_moe, made.values, made.scales, ids, weights, staged, dtype=torch.float32)
    want = HipExpertBackend(x_group="token", gu_dtype=torch.float32).forward_pairs(
        made.dequantize(torch.float32), ids[:, None], weights[:, None], staged)
    # a row's largest value is 448 scales, so its scale is found again but for its last bits; the hidden rows' codes may
    # each lie a step apart, 2^-3 of a value, in few of 256
    assert (got - want).abs().max() <= 2e-2 * want.abs().max()
    for row in (0, rows - 1):  # one row for several pairs
        a = fp8_decode.quantized_pairs(fp8_moe, made.values[row:row + 1], made.scales[row:row + 1], ids[row].expand(4),
                                       weights[row].expand(4), staged, dtype=torch.float32)
        assert torch.equal(a, a[:1].expand(4, HIDDEN))
        assert (a[0] - got[row]).abs().max() <= 2e-2 * got[row].abs().max()


@pytest.mark.parametrize("quant", ["fp8", "fp8-128"])
@pytest.mark.parametrize("tokens,top_k", [(1, 8), (3, 1), (3, 8), (20, 4), (37, 8), (500, 4), (777, 6)])
def test_a_prompts_rows_reach_their_experts_without_copies(cuda, tokens, top_k, quant):
    """ids [T, k] take row t for its k pairs: the bits of a call on rows that were repeated k times."""
    print_case("prompt's rows before experts", tokens, top_k, quant)
    g = torch.Generator().manual_seed(tokens)
    staged = bank(cuda)
    x = torch.randn(tokens, HIDDEN, generator=g).half().to(cuda)
    weight = (torch.rand(HIDDEN, generator=g) + 0.5).half().to(cuda)
    made = rms_norm(x, weight, residual=x, quant=quant).quant
    ids, weights = (t.reshape(tokens, top_k) for t in routes(tokens * top_k, g, cuda))
    got = fp8_decode.quantized_pairs(fp8_moe, made.values, made.scales, ids, weights, staged)
    assert got.shape == (tokens * top_k, HIDDEN)
    repeat = made.values.view(torch.uint8).repeat_interleave(top_k, 0).view(FP8_DTYPE), made.scales.repeat_interleave(top_k, 0)
    want = fp8_decode.quantized_pairs(fp8_moe, *repeat, ids.flatten(), weights.flatten(), staged)
    assert torch.equal(got, want)


@pytest.mark.parametrize("quant", ["fp8", "fp8-128"])
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_a_layers_norm_router_and_experts(cuda, tokens, quant):
    """One norm for router and experts: the sum of a prompt's partials is what the experts make of the held values."""
    print_case("norm, router and experts", tokens, quant)
    g = torch.Generator().manual_seed(tokens + 7)
    staged = bank(cuda)
    x, add = (torch.randn(tokens, HIDDEN, generator=g).bfloat16().to(cuda) for _ in range(2))
    made = rms_norm(x, (torch.rand(HIDDEN, generator=g) + 0.5).bfloat16().to(cuda), residual=add, quant=quant, rows=True)
    router = torch.randn(EXPERTS, HIDDEN, generator=g).bfloat16().to(cuda)
    weights, ids = torch.softmax(made.rows.float() @ router.float().T, -1).topk(4)
    partials = fp8_decode.quantized_pairs(fp8_moe, made.quant.values, made.quant.scales, ids, weights, staged,
                                          dtype=torch.float32)
    out = partials.view(*ids.shape, -1).sum(1)
    backend = HipExpertBackend(x_group="token" if quant == "fp8" else 128, gu_dtype=torch.float32)
    want = backend.forward(made.quant.dequantize(torch.float32), ids, weights, staged)
    # the held values are quantized to themselves but for their scales' last bits; hidden codes may lie a step apart
    assert (out - want).abs().max() <= 2e-2 * want.abs().max()
