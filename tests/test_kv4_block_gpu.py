"""GPU: a decoder layer over the 4-bit cache -- projections, append, attention,
output projection, MoE block -- as prompts and as captured decode steps."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_reference as ref
from conftest import print_case
from drama_moe.attention import KvCache4, PagedBatch, Rotary
from drama_moe.block import AttentionBlock, MoeBlock
from drama_moe.formats import StagedExperts, random_fp8_bank
from drama_moe.offload import HipExpertBackend
from drama_moe.quantized import GPTQLinear

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -7  # bf16


def wide(t):
    return t.detach().double().cpu().numpy()


class Layer:
    def __init__(self, cuda, *, hidden=512, heads=8, kv_heads=2, dim=128, page=32, pages=40, experts=16, seed=0, window=0):
        g = torch.Generator().manual_seed(seed)
        self.hidden, self.heads, self.kv_heads, self.dim = hidden, heads, kv_heads, dim

        def linear(k, n):
            words = torch.randint(-2 ** 31, 2 ** 31 - 1, (k // 8, n), generator=g).int()
            scales = (torch.rand(k // 128, n, generator=g) * 0.5 + 0.75).half() * (0.2 * k ** -0.5)
            return GPTQLinear(words, scales.half(), device=cuda)

        self.cache = KvCache4.allocate(pages, kv_heads, dim, page_size=page, device=cuda)
        self.inv_freq = (10000.0 ** (-np.arange(dim // 2) / (dim // 2))).astype(np.float32)
        self.axis = Rotary.sections([dim // 4, dim // 8, dim // 8], cyclic=True, device=cuda)
        self.attention = AttentionBlock(
            linear(hidden, heads * dim), linear(hidden, kv_heads * dim), linear(hidden, kv_heads * dim),
            linear(heads * dim, hidden), self.cache, heads=heads, window=window,
            rotary=Rotary(torch.from_numpy(self.inv_freq).to(cuda), axis=self.axis))
        w = lambda *shape: (torch.randn(*shape, generator=g) * 0.05).bfloat16().to(cuda)  # noqa: E731
        bank = random_fp8_bank(experts, hidden, 256, layout="channel", generator=g)
        staged = StagedExperts(*(getattr(bank, n).to(cuda) for n in ("w13_weight", "w13_scale_inv", "w2_weight",
                                                                     "w2_scale_inv")))
        self.moe = MoeBlock(w(experts, hidden), w(1, hidden), w(128, hidden), w(128, hidden), w(hidden, 128), staged,
                            HipExpertBackend(), top_k=4)

    def __call__(self, x, batch, positions):
        """x + attention(x), then the MoE half of that."""
        after = self.attention(x, x, batch, positions)
        return self.moe(after, after)[0]


def i32(cuda, *x):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("window", [0, 50])
def test_attention_half_against_the_reference(cuda, window):
    """Two prompts and a sequence of one row: the block is its parts, and they are what 64 bits say."""
    print_case("kv4 layer", window)
    layer = Layer(cuda, seed=1 + window, window=window)
    block, dim = layer.attention, layer.dim
    g = torch.Generator().manual_seed(2)
    seqs = [(90, 90), (1, 1), (33, 33)]
    rows = sum(n for n, _ in seqs) + 2
    x = torch.randn(rows, layer.hidden, generator=g).bfloat16().to(cuda)
    residual = torch.randn(rows, layer.hidden, generator=g).bfloat16().to(cuda)
    positions = torch.randint(0, 5000, (3, rows), generator=g)
    table = torch.randperm(40, generator=g)[:9].reshape(3, 3).int()
    starts = [0, 90, 91, 124]
    batch = PagedBatch(table.to(cuda), i32(cuda, 90, 1, 33), i32(cuda, *starts), rows=rows, max_rows=90)
    layer.cache.status()
    out = block(x, residual, batch, positions.to(cuda))
    assert out.dtype == torch.bfloat16 and out.shape == x.shape and layer.cache.status() == 0
    pages = layer.cache.pages.clone()

    # the parts by themselves: the same pages, and the block's output to the bit
    q, k, v = (proj(x).reshape(rows, -1, dim) for proj in (block.q_proj, block.k_proj, block.v_proj))
    layer.cache.pages.zero_()
    turned = layer.cache.append(k, v, batch, rotary=block.rotary, positions=positions.to(cuda), q=q)
    assert torch.equal(layer.cache.pages, pages)
    attended = torch.zeros(rows, layer.heads, dim, dtype=torch.bfloat16, device=cuda)
    layer.cache.attend(turned, batch, window=window, out=attended)
    assert torch.equal(out, residual + block.o_proj(attended.reshape(rows, -1)))
    assert torch.equal(out[124:], residual[124:])

    # and in 64 bits, from what the projections gave
    held = ref.Pages(torch.zeros_like(pages).cpu().numpy(), 32, dim)
    axis = layer.axis.cpu().numpy()
    keys = ref.rotate(wide(k), positions.numpy(), layer.inv_freq, axis, False).astype(np.float32)
    for s, (n, length) in enumerate(seqs):
        at = slice(starts[s], starts[s] + n)
        for p in range(length):
            held.put(int(table[s, p // 32]), p % 32, keys[at][p], wide(v)[at][p])
        kk, vv = held.tokens(table[s].tolist(), length)
        want, size, terms = ref.attention(wide(turned)[at], kk, vv, length, dim ** -0.5, window)
        bound = ref.tolerance(want, size, terms, dim, length, EPS)
        assert (np.abs(wide(attended)[at] - want) <= bound).all(), s
    assert np.array_equal(held.raw, pages.cpu().numpy())


def test_layer_in_prompts_then_captured_decode_steps(cuda):
    """Prompt, then steps by a graph of the whole layer: each the eager layer's, on a cache of the same contents."""
    print_case("kv4 layer decode")
    layer = Layer(cuda, seed=3)
    g = torch.Generator().manual_seed(4)
    n, longest = 3, 70
    table = torch.randperm(40, generator=g)[:12].reshape(n, 4).int().to(cuda)
    sizes = [70, 1, 40]
    prompt = PagedBatch(table, i32(cuda, *sizes), i32(cuda, 0, 70, 71, 111), rows=111, max_rows=longest)
    place = torch.cat([torch.arange(s) for s in sizes]).expand(3, -1).contiguous().to(cuda)
    first = layer(torch.randn(111, layer.hidden, generator=g).bfloat16().to(cuda), prompt, place)
    assert torch.isfinite(first.float()).all()

    lengths = i32(cuda, *sizes) + 1
    batch = PagedBatch(table, lengths)
    x = torch.zeros(n, layer.hidden, dtype=torch.bfloat16, device=cuda)
    positions = torch.zeros(3, n, dtype=torch.int64, device=cuda)
    side = torch.cuda.Stream(cuda)
    kept = layer.cache.pages.clone()
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        layer(x, batch, positions)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = layer(x, batch, positions)
    layer.cache.pages.copy_(kept)
    for step in range(6):
        x.copy_(torch.randn(n, layer.hidden, generator=g).bfloat16())
        positions.copy_((lengths - 1).long().expand(3, n))
        before = layer.cache.pages.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed, pages = out.clone(), layer.cache.pages.clone()
        layer.cache.pages.copy_(before)
        eager = layer(x, batch, positions)
        assert torch.equal(replayed, eager) and torch.equal(layer.cache.pages, pages), step
        assert not torch.equal(before, pages)
        lengths += 1
    assert layer.cache.status() == 0


def test_projections_that_need_gradients_are_refused(cuda):
    print_case("kv4 layer gradients")
    cache = KvCache4.allocate(8, 2, 64, page_size=16, device=cuda)
    linear = lambda k, n: torch.nn.Linear(k, n, bias=False, device=cuda, dtype=torch.float16)  # noqa: E731
    block = AttentionBlock(linear(64, 256), linear(64, 128), linear(64, 128), linear(256, 64), cache, heads=4)
    x = torch.randn(20, 64, device=cuda, dtype=torch.float16)
    batch = PagedBatch(i32(cuda, 3, 5).reshape(1, 2), i32(cuda, 20), i32(cuda, 0, 20), rows=20)
    with pytest.raises(ValueError, match="k needs gradients"):
        block(x, x, batch)
    assert not cache.pages.any()
    with torch.no_grad():
        assert torch.isfinite(block(x, x, batch)).all()
    for p in (block.q_proj, block.k_proj, block.v_proj):
        p.requires_grad_(False)
    out = block(x, x, batch)  # the output projection alone learns, which its own backward serves
    out.float().sum().backward()
    assert block.o_proj.weight.grad is not None


def test_norms_plain_linears_and_no_rotation(cuda):
    print_case("kv4 layer linears")
    torch.manual_seed(9)
    hidden, heads, kv, dim = 96, 6, 3, 64
    cache = KvCache4.allocate(8, kv, dim, page_size=16, device=cuda)
    linear = lambda k, n: torch.nn.Linear(k, n, bias=False, device=cuda, dtype=torch.float16)  # noqa: E731
    half = lambda t: (t * 0.5)  # noqa: E731
    projections = linear(hidden, heads * dim), linear(hidden, kv * dim), linear(hidden, kv * dim), linear(heads * dim, hidden)
    block = AttentionBlock(*projections, cache, heads=heads, q_norm=half, k_norm=half, scale=0.5)
    x = torch.randn(20, hidden, device=cuda, dtype=torch.float16)
    batch = PagedBatch(i32(cuda, 3, 5).reshape(1, 2), i32(cuda, 20), i32(cuda, 0, 20), rows=20)
    with torch.no_grad():
        out = block(x, x, batch)
        q, k, v = (p(x).reshape(20, -1, dim) for p in projections[:3])
        pages = cache.pages.clone()
        cache.append(k * 0.5, v, batch)
        assert torch.equal(cache.pages, pages)
        want = x + projections[3](cache.attend(q * 0.5, batch, scale=0.5).reshape(20, -1))
    assert torch.equal(out, want)
    empty = PagedBatch(i32(cuda, 3, 5).reshape(1, 2), i32(cuda, 20), i32(cuda, 0, 0), rows=0)
    with torch.no_grad():
        assert block(x[:0], x[:0], empty).shape == (0, hidden)
    with pytest.raises(ValueError, match="attn_input and residual"):
        block(x, x[:3], batch)
    with pytest.raises(ValueError, match="need a rotary"):
        block(x, x, batch, torch.arange(20, device=cuda))
