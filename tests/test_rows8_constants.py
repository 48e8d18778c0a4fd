"""Norms and products in 8 bits on the CPU: inputs whose gradients or tangents
the calls would lose, modules under casts, scales of quantized matrices."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import rows8_reference as ref
from drama_moe.attention import KvCache4, PagedBatch
from drama_moe.block import AttentionBlock
from drama_moe.int8 import Int8FeedForward, Int8Linear, Int8Weight, QuantRows, int8_feed_forward, int8_linear, quantize_rows
from drama_moe.norm import rms_norm
from drama_moe.quantized import GPTQLinear


def i8(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def weight(n=4, k=32):
    return Int8Weight(i8(n, k) + 1, torch.ones(n))


@pytest.mark.parametrize("name,call", [
    ("x", lambda d: quantize_rows(d(2, 32))),
    ("x", lambda d: int8_linear(d(2, 32), weight())),
    ("bias", lambda d: int8_linear(torch.zeros(2, 32), weight(), bias=d(4))),
    ("residual", lambda d: int8_linear(torch.zeros(2, 32), weight(), residual=d(2, 4))),
    ("bias", lambda d: int8_linear(QuantRows(i8(2, 32), torch.ones(2)), weight(), bias=d(4))),
    ("x", lambda d: int8_feed_forward(d(2, 32), weight(8), weight(5, 4))),
    ("residual", lambda d: int8_feed_forward(torch.zeros(2, 32), weight(8), weight(5, 4), residual=d(2, 5))),
    ("x", lambda d: rms_norm(d(2, 32), torch.ones(32))),
    ("weight", lambda d: rms_norm(torch.zeros(2, 32), d(32))),
    ("residual", lambda d: rms_norm(torch.zeros(2, 32), torch.ones(32), residual=d(2, 32))),
    ("scales", lambda d: QuantRows(i8(2, 32), d(2))),
    ("scales", lambda d: Int8Weight(i8(4, 32), d(4))),
    ("x", lambda d: Int8Linear(i8(4, 32), torch.ones(4))(d(2, 32))),
])
def test_forward_mode_tangents_are_refused(name, call):
    """A dual tensor has requires_grad false, and torch.no_grad() keeps its tangent."""
    with forward_ad.dual_level():
        dual = lambda *shape: forward_ad.make_dual(torch.zeros(shape), torch.ones(shape))  # noqa: E731
        with pytest.raises(ValueError, match=f"{name} has a forward-mode tangent"):
            call(dual)
        with torch.no_grad(), pytest.raises(ValueError, match=f"{name} has a forward-mode tangent"):
            call(dual)
        with torch.inference_mode():  # drops tangents: so does the call
            try:
                call(dual)
            except RuntimeError as e:
                assert "ROCm GPU" in str(e)
    with pytest.raises(ValueError, match="forward-mode tangent"):
        torch.func.jvp(lambda x: quantize_rows(x), (torch.zeros(2, 32),), (torch.ones(2, 32),))


def test_attention_block_refuses_forward_mode_tangents():
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device="cpu")
    batch = PagedBatch(torch.ones(2, 2).int(), torch.ones(2).int())
    linear = [torch.nn.Linear(32, 256), torch.nn.Linear(32, 128), torch.nn.Linear(32, 128), torch.nn.Linear(256, 32)]
    block = AttentionBlock(*linear, cache, heads=4)
    with torch.no_grad(), forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(2, 32), torch.ones(2, 32))
        with pytest.raises(ValueError, match="attn_input has a forward-mode tangent"):
            block(x, torch.zeros(2, 32), batch)


@pytest.mark.parametrize("cols", [32, 128])
def test_e4m3_values_that_need_gradients_are_refused(cols):
    values = torch.zeros(2, cols).to(torch.float8_e4m3fn).requires_grad_()
    with pytest.raises(ValueError, match="values needs gradients"):
        QuantRows(values, torch.ones(2))
    with torch.no_grad():
        QuantRows(values, torch.ones(2))


CASTS = {"bf16": lambda m: m.to(torch.bfloat16), "half": lambda m: m.half(), "double": lambda m: m.double(),
         "type": lambda m: m.type(torch.float16), "both": lambda m: m.to("cpu", torch.float16)}


@pytest.mark.parametrize("cast", CASTS)
def test_casts_of_a_layer_leave_the_types_of_its_buffers(cast):
    torch.manual_seed(0)
    linear = Int8Linear.from_linear(torch.nn.Linear(40, 24))
    bare = lambda k, n: torch.nn.Linear(k, n, bias=False)  # noqa: E731
    ffn = Int8FeedForward.from_linears(bare(24, 40), bare(24, 40), bare(40, 24))
    before = {n: t.clone() for m in (linear, ffn) for n, t in m.state_dict().items()}
    layer = torch.nn.Sequential(linear, torch.nn.Linear(3, 3), ffn)
    CASTS[cast](layer)
    assert layer[1].weight.dtype is (torch.float64 if cast == "double" else torch.bfloat16 if cast == "bf16" else torch.float16)
    after = {n: t for m in (linear, ffn) for n, t in m.state_dict().items()}
    assert before.keys() == after.keys()
    for n, t in before.items():
        assert after[n].dtype is t.dtype and torch.equal(after[n], t), n
    for m in (linear, ffn.gate_up, ffn.down):
        assert torch.equal(m._weight().values, m.qweight[:, :m.in_features])


def test_a_cast_of_a_layer_still_moves_its_buffers():
    linear = Int8Linear.from_linear(torch.nn.Linear(40, 24)).to("meta", torch.bfloat16)
    assert {t.device.type for t in linear.buffers()} == {"meta"}
    assert linear.scales.dtype is linear.bias.dtype is torch.float32 and linear.qweight.dtype is torch.int8


@pytest.mark.parametrize("cast", CASTS)
def test_casts_of_a_gptq_linear_leave_its_codes_and_scales(cast):
    """Its kernel reads fp16 scales: bits of another type would be taken for them."""
    linear = GPTQLinear(torch.arange(32 * 48, dtype=torch.int32).reshape(32, 48), torch.rand(2, 48).half(), device="cpu")
    codes, scales = linear.qweight.clone(), linear.scales.clone()
    CASTS[cast](torch.nn.Sequential(linear))
    assert linear.scales.dtype is torch.float16 and torch.equal(linear.scales, scales)
    assert linear.qweight.dtype is torch.int32 and torch.equal(linear.qweight, codes)
    assert linear.weight.dtype is (torch.float64 if cast == "double" else torch.bfloat16 if cast == "bf16" else torch.float16)


def test_scales_of_a_matrix_are_those_of_rows():
    """Largest magnitudes times fl32(1/127), which a division by 127 misses by a last bit in one row of twenty."""
    w = torch.randn(4000, 40, generator=torch.Generator().manual_seed(3))
    w[7] = 0
    held = Int8Weight.quantize(w)
    codes, scales = ref.int8(ref.wide(w))
    assert np.array_equal(ref.wide(held.scales), scales) and np.array_equal(ref.wide(held.values), codes)
    assert (held.scales != w.abs().amax(1).clamp(min=1e-12) / 127).float().mean() > 0.02


def test_a_linear_of_integers_leaves_the_float_one_alone():
    """State loaded into the one made of a float linear does not reach that linear's bias."""
    linear = torch.nn.Linear(40, 24)
    before = linear.bias.detach().clone()
    made = Int8Linear.from_linear(linear)
    assert torch.equal(made.bias, before)
    made.load_state_dict(Int8Linear.from_linear(torch.nn.Linear(40, 24)).state_dict())
    assert torch.equal(linear.bias, before) and not torch.equal(made.bias, before)
