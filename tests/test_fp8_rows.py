"""Rows in E4M3 handed to the FP8 experts, on the CPU: what
``fp8_decode.quantized_pairs`` refuses before any launch."""
import pytest
import torch

from drama_moe import fp8_decode, fp8_moe
from drama_moe.formats import FP8_DTYPE, random_fp8_bank

HIDDEN = 256


@pytest.fixture(scope="module")
def bank():
    return random_fp8_bank(4, HIDDEN, 128, generator=torch.Generator().manual_seed(5))


def rows(count, cols=HIDDEN):
    return torch.zeros(count, cols, dtype=torch.uint8).view(FP8_DTYPE)


def call(bank, q=None, scales=None, ids=None, weights=None):
    return fp8_decode.quantized_pairs(fp8_moe, rows(3) if q is None else q, torch.ones(3) if scales is None else scales,
                                      torch.zeros(3, dtype=torch.int64) if ids is None else ids,
                                      torch.ones(3) if weights is None else weights, bank)


@pytest.mark.parametrize("inputs,message", [
    (dict(scales=torch.ones(2)), "scales must be fp32 \\[rows\\] or \\[rows, 2\\]"),
    (dict(scales=torch.ones(3, 3)), "scales must be"),
    (dict(scales=torch.ones(2, 2)), "scales must be"),
    (dict(scales=torch.ones(3, 2, 1)), "scales must be"),
    (dict(scales=torch.ones(3).double()), "scales must be"),
    (dict(q=rows(2), scales=torch.ones(2)), "one shared row or one per pair"),
    (dict(q=rows(2), scales=torch.ones(2), ids=torch.zeros(3, 2, dtype=torch.int64), weights=torch.ones(3, 2)), "each row of ids"),
    (dict(ids=torch.zeros(3, 2, dtype=torch.int64)), "one weight per pair"),
    (dict(q=rows(3, 128)), "rows must be FP8 \\[rows, 256\\]"),
    (dict(q=rows(3, 512)[:, ::2]), "contiguous columns"),
    (dict(q=rows(3).float()), "rows must be FP8"),
    (dict(q=rows(3)[0]), "rows must be FP8"),
    (dict(weights=torch.ones(2)), "one weight per pair"),
    (dict(weights=torch.ones(3, device="meta")), "share a device"),
])
def test_refusals(bank, inputs, message):
    with pytest.raises(ValueError, match=message):
        call(bank, **inputs)


def test_no_pairs_are_no_launch(bank):
    none = torch.zeros(0, 4, dtype=torch.int64)
    assert call(bank, q=rows(0), scales=torch.ones(0), ids=none, weights=none.float()).shape == (0, HIDDEN)
    assert call(bank, q=rows(1), scales=torch.ones(1), ids=none, weights=none.float()).shape == (0, HIDDEN)
    assert call(bank, ids=none.reshape(3, 0), weights=none.reshape(3, 0).float()).shape == (0, HIDDEN)
