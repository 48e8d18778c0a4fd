"""GPU: norm, attention half and dense half of a decoder layer on 8-bit
integers, as prompts and as captured decode steps; the norm before a mixture
of experts; calls on other streams, in graphs captured apart, and repeated."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rows8_reference as ref
from conftest import print_case
from drama_moe import fp8_decode, fp8_moe
from drama_moe.attention import KvCache4, PagedBatch, Rotary
from drama_moe.block import AttentionBlock, DenseBlock, MoeBlock
from drama_moe.formats import StagedExperts, random_fp8_bank
from drama_moe.int8 import Int8FeedForward, Int8Linear, Int8Weight, int8_feed_forward, int8_linear, quantize_rows
from drama_moe.norm import RmsNorm, rms_norm
from drama_moe.offload import HipExpertBackend

pytestmark = pytest.mark.gpu


def i32(cuda, *x):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


class Layer:
    """norm -> attention half -> norm -> feed-forward, all products in 8 bits."""

    def __init__(self, cuda, *, hidden=512, heads=8, kv=2, dim=64, inter=700, seed=0):
        torch.manual_seed(seed)
        self.hidden, self.heads, self.dim = hidden, heads, dim
        make = lambda k, n: Int8Linear.from_linear(torch.nn.Linear(k, n), device=cuda)  # noqa: E731
        self.cache = KvCache4.allocate(48, kv, dim, page_size=16, device=cuda)
        rotary = Rotary((10000.0 ** (-torch.arange(dim // 2) / (dim // 2))).float().to(cuda))
        self.attention = AttentionBlock(make(hidden, heads * dim), make(hidden, kv * dim), make(hidden, kv * dim),
                                        make(heads * dim, hidden), self.cache, heads=heads, rotary=rotary)
        self.norm = RmsNorm((torch.rand(hidden) + 0.5).bfloat16().to(cuda), quant="int8")
        bare = lambda k, n: torch.nn.Linear(k, n, bias=False)  # noqa: E731
        self.dense = DenseBlock(RmsNorm((torch.rand(hidden) * 0.2).bfloat16().to(cuda), offset=1.0, quant="int8"),
                                Int8FeedForward.from_linears(bare(hidden, inter), bare(hidden, inter), bare(inter, hidden),
                                                             device=cuda))

    def __call__(self, x, batch, positions=None):
        return self.dense(self.attention(self.norm(x).quant, x, batch, positions))


def test_layer_is_its_parts(cuda):
    """A prompt through the layer: each part against 64 bits on what the part before it gave."""
    print_case("dense layer parts")
    layer = Layer(cuda, seed=1)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(90, 512, generator=g).bfloat16().to(cuda)
    table = torch.randperm(48, generator=g)[:6].reshape(1, 6).int().to(cuda)
    batch = PagedBatch(table, i32(cuda, 90), i32(cuda, 0, 90), rows=90)
    out = layer(x, batch)
    pages = layer.cache.pages.clone()

    made = layer.norm(x)
    _, y = ref.norm(ref.wide(x), None, ref.wide(layer.norm.weight), torch.bfloat16, eps=1e-6)
    codes, scales = ref.int8(y)
    assert np.array_equal(ref.wide(made.quant.values.float()), codes) and np.array_equal(ref.wide(made.quant.scales), scales)
    a = layer.attention
    q, k, v = (p(made.quant) for p in (a.q_proj, a.k_proj, a.v_proj))
    for t, p in ((q, a.q_proj), (k, a.k_proj), (v, a.v_proj)):
        want, size = ref.product(codes, scales, ref.wide(p.qweight), ref.wide(p.scales), ref.wide(p.bias))
        slack = 6 * 2.0 ** -24 * size
        assert (np.abs(ref.wide(t) - want) <= slack + 2.0 ** -8 * (np.abs(want) + slack)).all()
    layer.cache.pages.zero_()
    turned = layer.cache.append(k.view(90, 2, 64), v.view(90, 2, 64), batch, rotary=a.rotary, q=q.view(90, 8, 64))
    assert torch.equal(layer.cache.pages, pages)
    attended = layer.cache.attend(turned, batch).reshape(90, 512)
    after = a.o_proj(attended, residual=x)
    c, s = ref.int8(ref.wide(attended))
    want, size = ref.product(c, s, ref.wide(a.o_proj.qweight), ref.wide(a.o_proj.scales), ref.wide(a.o_proj.bias), ref.wide(x))
    slack = 6 * 2.0 ** -24 * size
    assert (np.abs(ref.wide(after) - want) <= slack + 2.0 ** -8 * (np.abs(want) + slack)).all()
    made = layer.dense.norm(after)
    up, down = layer.dense.ffn.gate_up, layer.dense.ffn.down
    assert torch.equal(out, layer.dense.ffn(made.quant, residual=after))
    _, y = ref.norm(ref.wide(after), None, ref.wide(layer.dense.norm.weight), torch.bfloat16, eps=1e-6, offset=1.0)
    low, high = ref.feed_forward(*ref.int8(y), ref.wide(up.qweight), ref.wide(up.scales), ref.wide(down.qweight)[:, :700],
                                 ref.wide(down.scales), torch.bfloat16, "silu", ref.wide(after))
    slack = 2.0 ** -8 * np.maximum(np.abs(low), np.abs(high))
    assert (ref.wide(out) >= low - slack).all() and (ref.wide(out) <= high + slack).all()


@pytest.mark.parametrize("seqs", [1, 3, 20])
def test_layer_in_captured_decode_steps(cuda, seqs):
    """Steps by a graph of the whole layer, eager steps between: each replay the eager layer's bits."""
    print_case("dense layer decode", seqs)
    layer = Layer(cuda, seed=3)
    g = torch.Generator().manual_seed(4)
    table = torch.randperm(48, generator=g)[:2 * seqs].reshape(seqs, 2).int().to(cuda)
    lengths = torch.randint(1, 20, (seqs,), generator=g).int().to(cuda)
    batch = PagedBatch(table, lengths)
    x = torch.zeros(seqs, layer.hidden, dtype=torch.bfloat16, device=cuda)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        layer(x, batch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = layer(x, batch)
    for step in range(5):
        x.copy_(torch.randn(seqs, layer.hidden, generator=g).bfloat16())
        before = layer.cache.pages.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed, pages = out.clone(), layer.cache.pages.clone()
        layer.cache.pages.copy_(before)
        eager = layer(x, batch)
        assert torch.equal(replayed, eager) and torch.equal(layer.cache.pages, pages), step
        lengths += 1
    assert layer.cache.status() == 0


def test_dense_block_adds_its_residual(cuda):
    print_case("dense block residual")
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        torch.manual_seed(5)
        bare = lambda k, n: torch.nn.Linear(k, n, bias=False)  # noqa: E731
        ffn = Int8FeedForward.from_linears(bare(96, 130), bare(96, 130), bare(130, 96), activation="gelu_tanh", device=cuda)
        x, r = torch.randn(2, 9, 96).to(cuda, dtype), torch.randn(2, 9, 96).to(cuda, dtype)
        for quant in (None, "int8"):
            norm = RmsNorm(torch.rand(96).to(cuda), quant=quant)
            block = DenseBlock(norm, ffn)
            h = x + r
            out = block(x, r)
            assert out.shape == x.shape and out.dtype is dtype and torch.equal(out, block(h))
            rows = rms_norm(h, norm.weight).rows
            if quant is None:  # the rows are rounded to their type before they are quantized
                assert torch.equal(out, int8_feed_forward(rows, ffn.gate_up._weight(), ffn.down._weight(),
                                                          activation="gelu_tanh", residual=h))
            made = rms_norm(h.reshape(18, 96), norm.weight, quant="int8").quant
            if quant:
                assert torch.equal(out.reshape(18, 96), ffn(made, residual=h.reshape(18, 96)))


def test_norm_before_a_mixture_of_experts(cuda):
    """One norm gives the router's rows and the experts' E4M3 groups, which the experts take as they are."""
    print_case("norm before experts")
    g = torch.Generator().manual_seed(6)
    hidden, experts = 512, 16
    w = lambda *shape: (torch.randn(*shape, generator=g) * 0.05).bfloat16().to(cuda)  # noqa: E731
    bank = random_fp8_bank(experts, hidden, 256, layout="block", generator=g)
    staged = StagedExperts(*(getattr(bank, n).to(cuda) for n in ("w13_weight", "w13_scale_inv", "w2_weight", "w2_scale_inv")))
    moe = MoeBlock(w(experts, hidden), w(1, hidden), w(128, hidden), w(128, hidden), w(hidden, 128), staged, HipExpertBackend(),
                   top_k=4)
    x, r = (torch.randn(5, hidden, generator=g).bfloat16().to(cuda) for _ in range(2))
    made = RmsNorm(w(hidden), offset=1.0)(x, r)
    out, weights, ids = moe(made.rows, made.hidden)
    assert torch.equal(made.hidden, x + r) and torch.isfinite(out.float()).all()
    both = rms_norm(x, torch.ones(hidden, device=cuda), residual=r, quant="fp8-128", rows=True)
    own, own_scales = fp8_moe.quantize_groups(fp8_moe.quant_kernel, both.rows, hidden)
    # The experts' quantizer sees the rows rounded to bf16, by at most 2^-8 of a value: so far the scales are apart.  A
    # held value is off by half a step, 2^-4 of the value (of a subnormal 2^-10 of the scale), from the row before that
    # rounding: (2^-4 + 2^-8) (1 + 2^-7) of the rounded one.
    assert ((both.quant.scales - own_scales).abs() <= own_scales * (2.0 ** -8 + 2.0 ** -22)).all()
    a, rows = both.quant.dequantize(torch.float32), both.rows.float()
    scale = both.quant.scales.repeat_interleave(128, 1)
    assert ((a - rows).abs() <= rows.abs() * (2.0 ** -4 + 2.0 ** -8) * (1 + 2.0 ** -7) + scale * 2.0 ** -10).all()
    for row in range(5):
        q, s = both.quant.values[row:row + 1], both.quant.scales[row:row + 1]
        got = fp8_decode.quantized_pairs(fp8_moe, q, s, ids[row], weights[row], staged)
        near = HipExpertBackend().forward(a[row:row + 1].bfloat16(), ids[row:row + 1], weights[row:row + 1], staged)
        assert (got.sum(0) - near[0].float()).abs().max() < 0.1 * near.float().abs().max()


def test_calls_on_other_streams_and_graphs_of_their_own(cuda):
    """Two streams at once, two graphs replayed in turn and at once: nothing is shared between calls."""
    print_case("dense streams and graphs")
    g = torch.Generator().manual_seed(7)
    make = lambda n, k: Int8Weight((torch.randn(n, k, generator=g) * 40).round().clamp(-128, 127).to(torch.int8).to(cuda),  # noqa: E731
                                   torch.rand(n, generator=g).to(cuda) * 0.001)
    up, down, deep = make(2 * 900, 1100), make(1100, 900), make(500, 9000)
    gain = torch.rand(1100, generator=g).to(cuda)

    def work(x, z):
        made = rms_norm(x, gain, residual=x, quant="int8")
        return int8_feed_forward(made.quant, up, down, residual=made.hidden, dtype=x.dtype), int8_linear(z, deep)

    inputs = [(torch.randn(rows, 1100, generator=g).bfloat16().to(cuda), torch.randn(rows, 9000, generator=g).half().to(cuda))
              for rows in (3, 40, 50, 64, 200)]
    plain = [work(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in inputs]
    for _ in range(4):
        got = []
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(work(*i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(plain, got) for a, b in zip(p, q))
    graphs, outs = [], []
    for s, i in zip(streams, inputs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            outs.append(work(*i))
    for turn in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            if turn % 2:
                with torch.cuda.stream(s):
                    graph.replay()
            else:
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(plain, outs) for a, b in zip(p, q)), turn
        assert all(torch.equal(a, b) for p, q in zip(plain, [work(*i) for i in inputs]) for a, b in zip(p, q))


def test_the_same_call_gives_the_same_bits(cuda):
    print_case("dense repeated")
    g = torch.Generator().manual_seed(8)
    w = Int8Weight((torch.randn(700, 5000, generator=g) * 40).round().clamp(-128, 127).to(torch.int8).to(cuda),
                   torch.rand(700, generator=g).to(cuda))
    for rows in (1, 30, 60, 300):
        x = torch.randn(rows, 5000, generator=g).to(cuda)
        first = int8_linear(x, w)
        assert all(torch.equal(first, int8_linear(x, w)) for _ in range(5))
        q = quantize_rows(x)
        assert torch.equal(int8_linear(q, w, dtype=torch.float32), first)


def test_memory_behind_the_operands_is_not_written_and_does_not_matter(cuda):
    """Rows, matrix and residual inside larger tensors whose other values are the lowest and highest of their types."""
    print_case("dense surroundings")
    g = torch.Generator().manual_seed(9)
    for rows, k, n in ((3, 33, 70), (20, 200, 33), (70, 130, 65), (300, 1000, 130)):
        width = -(-k // 16) * 16
        held = torch.full((n + 2, width + 16), -128, dtype=torch.int8, device=cuda)
        codes = (torch.randn(n, k, generator=g) * 40).round().clamp(-128, 127).to(torch.int8).to(cuda)
        held[1:n + 1, :k] = codes
        scales = torch.rand(n, generator=g).to(cuda)
        room = torch.full((rows + 2, k + 8), float("inf"), dtype=torch.bfloat16, device=cuda)
        x = torch.randn(rows, k, generator=g).bfloat16().to(cuda)
        room[1:rows + 1, 3:3 + k] = x
        add = torch.full((rows + 2, n + 5), float("nan"), dtype=torch.bfloat16, device=cuda)
        add[1:rows + 1, 2:2 + n] = 1.0
        before = held.clone(), room.clone()
        got = int8_linear(room[1:rows + 1, 3:3 + k], Int8Weight(held[1:n + 1, :k], scales), residual=add[1:rows + 1, 2:2 + n])
        want = int8_linear(x, Int8Weight(codes, scales), residual=torch.ones(rows, n, dtype=torch.bfloat16, device=cuda))
        assert torch.equal(got, want) and torch.isfinite(got.float()).all()
        assert torch.equal(held, before[0]) and torch.equal(room, before[1])
        made = rms_norm(room[1:rows + 1, 3:3 + k], torch.ones(k, device=cuda), quant="int8", rows=True)
        same = rms_norm(x, torch.ones(k, device=cuda), quant="int8", rows=True)
        assert torch.equal(made.rows, same.rows) and torch.equal(made.quant.values, same.quant.values)


def test_inputs_that_need_gradients_are_refused_unless_gradients_are_off(cuda):
    print_case("dense gradients")
    w = Int8Weight(torch.ones(4, 32, dtype=torch.int8, device=cuda), torch.ones(4, device=cuda))
    x = torch.randn(2, 32, device=cuda, requires_grad=True)
    with pytest.raises(ValueError, match="x needs gradients"):
        int8_linear(x, w)
    with pytest.raises(ValueError, match="x needs gradients"):
        rms_norm(x, torch.ones(32, device=cuda))
    with torch.no_grad():
        assert int8_linear(x, w).shape == (2, 4)


def test_tensors_of_two_devices_and_shapes_are_refused(cuda):
    print_case("dense devices")
    w = Int8Weight(torch.ones(4, 32, dtype=torch.int8, device=cuda), torch.ones(4, device=cuda))
    x = torch.randn(2, 32, device=cuda)
    for bad, message in ((dict(bias=torch.ones(4)), "bias must be on"), (dict(residual=torch.ones(2, 4)), "residual must be on"),
                         (dict(bias=torch.ones(3, device=cuda)), "bias must be fp32"),
                         (dict(bias=torch.ones(4, device=cuda).half()), "bias must be fp32"),
                         (dict(residual=torch.ones(2, 5, device=cuda)), "residual must be"),
                         (dict(residual=torch.ones(4, device=cuda)), "residual must be")):
        with pytest.raises(ValueError, match=message):
            int8_linear(x, w, **bad)
    with pytest.raises(ValueError, match="x must be on"):
        int8_linear(x.cpu(), w)
    with pytest.raises(ValueError, match="weight must be on"):
        rms_norm(x, torch.ones(32))
    with pytest.raises(ValueError, match="down must be on"):
        int8_feed_forward(x, Int8Weight(torch.ones(8, 32, dtype=torch.int8, device=cuda), torch.ones(8, device=cuda)),
                          Int8Weight(torch.ones(4, 4, dtype=torch.int8), torch.ones(4)))
    empty = int8_feed_forward(x[:0], Int8Weight(torch.ones(8, 32, dtype=torch.int8, device=cuda), torch.ones(8, device=cuda)), w.__class__(
        torch.ones(5, 4, dtype=torch.int8, device=cuda), torch.ones(5, device=cuda)))
    assert empty.shape == (0, 5) and quantize_rows(x[:0]).dequantize().shape == (0, 32)
