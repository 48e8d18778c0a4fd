"""GPU: tensors with a forward-mode tangent are refused where it would be
lost, as inputs that need gradients are."""
import pytest
import torch
from torch.autograd import forward_ad

from conftest import print_case
from drama_moe.attention import KvCache4, PagedBatch
from drama_moe.int8 import Int8Weight, QuantRows, int8_feed_forward, int8_linear, quantize_rows
from drama_moe.norm import rms_norm

pytestmark = pytest.mark.gpu


def test_forward_mode_tangents_are_refused(cuda):
    print_case("forward-mode tangents")
    i8 = lambda n, k: torch.ones(n, k, dtype=torch.int8, device=cuda)  # noqa: E731
    w, up, down = (Int8Weight(i8(n, k), torch.ones(n, device=cuda)) for n, k in ((4, 32), (8, 32), (5, 4)))
    x, gain = torch.randn(2, 32, device=cuda), torch.ones(32, device=cuda)
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device=cuda)
    batch = PagedBatch(torch.tensor([[0, 1], [2, 3]], device=cuda).int(), torch.tensor([1, 1], device=cuda).int())
    heads = lambda n: torch.randn(2, n, 64, device=cuda).bfloat16()  # noqa: E731
    k, v, q = heads(2), heads(2), heads(4)
    calls = {
        "x": [lambda t: quantize_rows(t(x)), lambda t: int8_linear(t(x), w), lambda t: int8_feed_forward(t(x), up, down),
              lambda t: rms_norm(t(x), gain)],
        "scales": [lambda t: QuantRows(i8(2, 32), t(gain[:2])), lambda t: Int8Weight(i8(4, 32), t(gain[:4]))],
        "weight": [lambda t: rms_norm(x, t(gain))],
        "k": [lambda t: cache.append(t(k), v, batch)],
        "v": [lambda t: cache.append(k, t(v), batch)],
        "q": [lambda t: cache.attend(t(q), batch)],
        "out": [lambda t: cache.attend(q, batch, out=t(torch.empty_like(q)))],
        "k_out": [lambda t: cache.read(batch, dtype=torch.bfloat16, k_out=t(torch.empty_like(k)))],
    }
    pages = cache.pages.clone()
    for name, each in calls.items():
        for call in each:
            with torch.no_grad(), forward_ad.dual_level():
                dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
                with pytest.raises(ValueError, match=f"{name} has a forward-mode tangent"):
                    call(dual)
                assert torch.equal(cache.pages, pages)
                primal = lambda t: forward_ad.unpack_dual(dual(t)).primal  # noqa: E731
                call(primal)  # what a tensor without a tangent gives, in a level too
                cache.pages.copy_(pages)
