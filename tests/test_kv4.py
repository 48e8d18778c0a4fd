"""The 4-bit paged cache on the CPU: what its Python classes and its C entry
points refuse before any GPU work, axis tables, and the reference that the GPU
tests use."""
from __future__ import annotations

import ctypes
import shutil
import subprocess

import numpy as np
import pytest
import torch

import kv4_reference as ref
from conftest import ROOT
from drama_moe import _lib
from drama_moe.attention import KvCache4, PagedBatch, Rotary
from drama_moe.block import AttentionBlock


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("make,message", [
    (lambda: PagedBatch(i32(2, 3).long(), i32(2)), "block_table must be int32"),
    (lambda: PagedBatch(i32(2, 3), i32(2).long()), "lengths must be int32"),
    (lambda: PagedBatch(i32(3, 3), i32(2)), "one entry a sequence"),
    (lambda: PagedBatch(i32(0, 3), i32(0)), "sequence count"),
    (lambda: PagedBatch(i32(4097, 1), i32(4097)), "sequence count"),
    (lambda: PagedBatch(i32(2, 0), i32(2)), "no pages"),
    (lambda: PagedBatch(i32(3, 2).T, i32(2)), "contiguous rows"),
    (lambda: PagedBatch(i32(2, 3), i32(2), i32(2), rows=4), r"starts must be \[sequences \+ 1\]"),
    (lambda: PagedBatch(i32(2, 3), i32(2), i32(3)), "rows is required"),
    (lambda: PagedBatch(i32(2, 3), i32(2), rows=1), "cover every sequence"),
    (lambda: PagedBatch(i32(2, 3), i32(2), i32(3), rows=4, max_rows=5), "max_rows outside"),
    (lambda: PagedBatch(i32(2, 3), i32(2), i32(3), rows=4, max_rows=0), "max_rows outside"),
    (lambda: PagedBatch(i32(2, 3), i32(2), i32(3), rows=2 ** 24 + 1), "row count"),
    (lambda: PagedBatch(i32(2, 3), i32(2), i32(3), rows=2 ** 32 + 6, max_rows=6), "row count"),
    (lambda: PagedBatch(i32(2, 3), i32(2), rows=2 ** 32 + 6), "row count"),
    (lambda: KvCache4(torch.zeros(4, 2, 16 * 72, dtype=torch.uint8), page_size=16, head_dim=80), "head_dim"),
    (lambda: KvCache4(torch.zeros(4, 2, 24 * 72, dtype=torch.uint8), page_size=24, head_dim=64), "power of two"),
    (lambda: KvCache4(torch.zeros(4, 2, 16 * 72 + 1, dtype=torch.uint8), page_size=16, head_dim=64), "pages must be"),
    (lambda: KvCache4(torch.zeros(4, 2, 16 * 72, dtype=torch.int8), page_size=16, head_dim=64), "pages must be"),
    (lambda: KvCache4(torch.zeros(0, 2, 16 * 72, dtype=torch.uint8), page_size=16, head_dim=64), "pages must be"),
    (lambda: KvCache4(torch.zeros(4, 4, 16 * 72, dtype=torch.uint8)[:, ::2], page_size=16, head_dim=64), "contiguous"),
    (lambda: KvCache4(torch.zeros(4, 2, 16 * 72 + 8, dtype=torch.uint8)[..., 8:], page_size=16, head_dim=64), "contiguous"),
    (lambda: Rotary(torch.ones(64, dtype=torch.float64)), "inv_freq must be"),
    (lambda: Rotary(torch.ones(12)), "multiple of 16"),
    (lambda: Rotary(torch.ones(0)), "multiple of 16"),
    (lambda: Rotary(torch.ones(16), axis=torch.zeros(8, dtype=torch.uint8)), "axis must be"),
    (lambda: Rotary(torch.ones(16), axis=torch.zeros(16, dtype=torch.int64)), "axis must be"),
    (lambda: Rotary.sections([]), "sections"),
    (lambda: Rotary.sections([4, -1]), "sections"),
])
def test_python_refusals(make, message):
    with pytest.raises(ValueError, match=message):
        make()


@pytest.mark.parametrize("seqs,cols,size,stride", [
    (3, 5, 5, 0), (2, 1, 1, 0), (4096, 2, 2, 0),          # one row for all: row.expand(seqs, cols)
    (1, 5, 5, 0), (1, 5, 5, 1), (1, 5, 5, 400),           # one sequence, whatever its row stride is
    (3, 5, 15, 5), (3, 5, 19, 7), (3, 1, 3, 1)])
def test_tables_are_read_where_they_lie(seqs, cols, size, stride):
    """The descriptor's places of all entries are those of the tensor."""
    table = torch.arange(size, dtype=torch.int32).as_strided((seqs, cols), (stride, 1))
    desc = PagedBatch(table, i32(seqs)).desc
    assert (desc.seqs, desc.table_cols) == (seqs, cols)
    places = np.arange(seqs)[:, None] * desc.table_stride + np.arange(cols)
    assert places.max() < size and np.array_equal(places, table.numpy())


@pytest.mark.parametrize("seqs,cols,stride", [(3, 5, 2), (2, 5, 4), (3, 2, 1)])
def test_tables_whose_rows_overlap_are_refused(seqs, cols, stride):
    table = i32((seqs - 1) * stride + cols).as_strided((seqs, cols), (stride, 1))
    with pytest.raises(ValueError, match="rows overlap"):
        PagedBatch(table, i32(seqs))


@pytest.mark.parametrize("stride,accepted", [(0, True), (1, False), (3, False), (4, True), (9, True)])
def test_entry_points_take_one_table_row_for_all_sequences(stride, accepted):
    cache, batch, _, _ = descriptors(batch=dict(table_stride=stride, block_table=None, lengths=None))
    size = _lib.library().dmoe_kv4_attention_workspace_bytes(ctypes.byref(cache), ctypes.byref(batch), 4)
    assert (size > 0) == accepted
    if not accepted:
        for entry in ("append", "read", "attend"):
            assert call(entry, descriptors(batch=dict(table_stride=stride))) == -1
            assert "block_table geometry" in _lib.library().dmoe_last_error().decode()


def test_there_is_no_cpu_path():
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device="cpu")
    batch = PagedBatch(i32(1, 2), i32(1))
    rows = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: cache.append(rows, rows, batch), lambda: cache.read(batch), lambda: cache.attend(rows, batch),
                 cache.status):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_axis_tables():
    assert Rotary.sections([3, 2, 1]).tolist() == [0, 0, 0, 1, 1, 2]
    assert Rotary.sections([3, 1, 2], cyclic=True).tolist() == [0, 1, 2, 0, 2, 0]
    assert Rotary.sections([2, 0, 1]).tolist() == [0, 0, 2]
    table = Rotary.sections([4, 2, 2])
    assert table.dtype == torch.uint8
    assert Rotary(torch.ones(8), axis=table).dim == 16


FAKE = 0x100000


def descriptors(cache=None, batch=None, rotary=None, rows=None):
    c = dict(pages=FAKE, page_stride=2 * 16 * 144, num_pages=8, page_size=16, kv_heads=2, head_dim=128) | (cache or {})
    b = dict(block_table=FAKE, table_stride=4, lengths=FAKE, starts=FAKE, seqs=2, table_cols=4, rows=6,
             max_rows=3) | (batch or {})
    r = dict(inv_freq=FAKE, axis=None, positions=FAKE, axis_stride=6, positions_dtype=_lib.I64, axes=2, dim=64,
             interleaved=0) | (rotary or {})
    h = dict(data=FAKE, row_stride=256, head_stride=128) | (rows or {})
    return _lib.Kv4Cache(**c), _lib.Kv4Batch(**b), _lib.RotaryDesc(**r), _lib.HeadRows(**h)


def call(entry, d, *, dtype=_lib.BF16, q_heads=4, scale=1.0, window=0, ws=FAKE, ws_bytes=1 << 40, q=None):
    lib, by = _lib.library(), ctypes.byref
    cache, batch, rotary, rows = d
    q = q or _lib.HeadRows(FAKE, q_heads * 128, 128)
    if entry == "append":
        return lib.dmoe_kv4_append(by(cache), by(batch), by(rotary), by(q), q_heads, by(q), by(rows), by(rows), dtype,
                                   None, None)
    if entry == "read":
        return lib.dmoe_kv4_read(by(cache), by(batch), by(rows), by(rows), dtype, None, None)
    return lib.dmoe_kv4_attention(by(cache), by(batch), by(q), q_heads, scale, window, by(q), dtype, ws, ws_bytes,
                                  None, None)


@pytest.mark.parametrize("entry", ["append", "read", "attend"])
@pytest.mark.parametrize("change,message", [
    (dict(cache=dict(pages=None)), "pages are required"),
    (dict(cache=dict(pages=FAKE + 8)), "16-byte aligned"),
    (dict(cache=dict(page_stride=2 * 16 * 144 + 8)), "16-byte aligned"),
    (dict(cache=dict(page_stride=16 * 144)), "smaller than a page"),
    (dict(cache=dict(head_dim=96)), "head_dim"),
    (dict(cache=dict(page_size=8)), "page_size"),
    (dict(cache=dict(page_size=48)), "page_size"),
    (dict(cache=dict(page_size=512)), "page_size"),
    (dict(cache=dict(num_pages=0)), "head count"),
    (dict(cache=dict(kv_heads=0)), "head count"),
    (dict(batch=dict(block_table=None)), "block_table and lengths"),
    (dict(batch=dict(lengths=None)), "block_table and lengths"),
    (dict(batch=dict(seqs=0)), "sequence count"),
    (dict(batch=dict(seqs=4097)), "sequence count"),
    (dict(batch=dict(rows=0)), "row count"),
    (dict(batch=dict(rows=(1 << 24) + 1)), "row count"),
    (dict(batch=dict(max_rows=0)), "max_rows"),
    (dict(batch=dict(max_rows=7)), "max_rows"),
    (dict(batch=dict(starts=None, rows=1, max_rows=1)), "one row a sequence"),
    (dict(batch=dict(table_cols=0)), "block_table geometry"),
    (dict(batch=dict(table_stride=3)), "block_table geometry"),
])
def test_entry_points_refuse_bad_descriptors(entry, change, message):
    assert call(entry, descriptors(**change)) == -1
    assert message in _lib.library().dmoe_last_error().decode()


@pytest.mark.parametrize("entry,change,kw,message", [
    ("append", dict(rotary=dict(inv_freq=None)), {}, "frequencies"),
    ("append", dict(rotary=dict(dim=24)), {}, "multiple of 16"),
    ("append", dict(rotary=dict(dim=144)), {}, "multiple of 16"),
    ("append", dict(rotary=dict(axes=0)), {}, "axis"),
    ("append", dict(rotary=dict(axis_stride=5)), {}, "axes overlap"),
    ("append", dict(rotary=dict(positions_dtype=_lib.F32)), {}, "int32 or int64"),
    ("append", dict(), dict(dtype=_lib.F32), "bf16 or fp16"),
    ("append", dict(rows=dict(data=None)), {}, "k rows are required"),
    ("append", dict(rows=dict(data=FAKE + 2)), {}, "k rows must have 16-byte aligned"),
    ("append", dict(rows=dict(row_stride=257)), {}, "16-byte aligned"),
    ("append", dict(rows=dict(head_stride=-128)), {}, "non-negative"),
    ("append", dict(rows=dict(row_stride=1 << 40)), {}, "too large"),
    ("append", dict(), dict(q_heads=0), "q_heads"),
    ("append", dict(), dict(q=_lib.HeadRows(FAKE, 128, 128)), "q_out rows overlap"),
    ("read", dict(), dict(dtype=_lib.I32), "bf16 or fp16"),
    ("read", dict(rows=dict(row_stride=128)), {}, "k_out rows overlap"),
    ("attend", dict(), dict(q_heads=3), "multiple of the key/value heads"),
    ("attend", dict(), dict(q_heads=0), "multiple of the key/value heads"),
    ("attend", dict(), dict(scale=0.0), "scale"),
    ("attend", dict(), dict(scale=-1.0), "scale"),
    ("attend", dict(), dict(scale=float("nan")), "scale"),
    ("attend", dict(), dict(scale=float("inf")), "scale"),
    ("attend", dict(), dict(window=-1), "window"),
    ("attend", dict(), dict(ws=None), "workspace too small"),
    ("attend", dict(batch=dict(table_cols=400, table_stride=400)), dict(ws_bytes=64), "workspace too small"),
    ("attend", dict(), dict(ws=FAKE + 8), "workspace must be 16-byte aligned"),
    ("attend", dict(), dict(q=_lib.HeadRows(FAKE, 512, 0)), "out rows overlap"),
])
def test_entry_points_refuse_bad_arguments(entry, change, kw, message):
    assert call(entry, descriptors(**change), **kw) == -1
    assert message in _lib.library().dmoe_last_error().decode()


def test_workspace_covers_more_rows_with_more_bytes():
    lib, by = _lib.library(), ctypes.byref
    sizes = []
    for rows, most in ((2, 1), (600, 300), (6000, 3000)):
        cache, batch, _, _ = descriptors(batch=dict(rows=rows, max_rows=most, block_table=None, lengths=None,
                                                    table_cols=900, table_stride=900))
        sizes.append(lib.dmoe_kv4_attention_workspace_bytes(by(cache), by(batch), 4))
    assert 0 < sizes[0] <= sizes[1] <= sizes[2]
    cache, batch, _, _ = descriptors(batch=dict(seqs=0))
    assert lib.dmoe_kv4_attention_workspace_bytes(by(cache), by(batch), 4) == 0
    cache, batch, _, _ = descriptors()
    assert lib.dmoe_kv4_attention_workspace_bytes(by(cache), by(batch), 5) == 0


@pytest.mark.parametrize("dim,kv_heads,heads", [(64, 4, 4), (128, 8, 32), (256, 2, 16)])
def test_workspace_is_bounded(dim, kv_heads, heads):
    """Room for partial sums of what can be cut: two for each of 256 workgroups' tiles of 128 or 256 rows and 2 (D + 2)
    fp32 at most, however many rows there are; for few rows no more than the table has blocks."""
    lib, by = _lib.library(), ctypes.byref

    def need(seqs, rows, most, cols):
        cache, batch, _, _ = descriptors(dict(page_stride=kv_heads * 16 * (dim + dim // 8), kv_heads=kv_heads, head_dim=dim),
                                         dict(seqs=seqs, rows=rows, max_rows=most, table_cols=cols, table_stride=cols))
        return lib.dmoe_kv4_attention_workspace_bytes(by(cache), by(batch), heads)

    tile = (128 if dim == 256 else 256) * (dim + 2) * 4
    for seqs, rows, most in ((1, 32768, 32768), (1, 131072, 131072), (40, 1 << 20, 100000)):
        assert 0 < need(seqs, rows, most, most // 16) <= 2 * 256 * tile
    for cols in (12, 44):  # a wave's share is two blocks of 64 tokens or more; each leaves two partial sums of 16 rows
        group = heads // kv_heads
        assert 0 < need(1, 1, 1, cols) <= 2 * kv_heads * -(-cols * 16 // 128) * 16 * (dim + 2) * 4 + kv_heads * 16, group


def places_check(tmp_path, header):
    (tmp_path / "kv4_places.hpp").write_text(header)
    exe = tmp_path / "places_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-Wall", "-Werror", "-I", str(tmp_path),
                    str(ROOT / "tests" / "kv4_places_check.cpp"), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_places_of_tokens_up_to_the_longest_sequence(tmp_path):
    header = (ROOT / "drama3-studio_amd" / "csrc" / "kv4_places.hpp").read_text()
    run = places_check(tmp_path, header)
    assert run.returncode == 0 and run.stdout.startswith("ok "), run.stdout + run.stderr
    # the check sees a place formed in 31 bits before it is cut
    signed = header.replace("const uint32_t token = (uint32_t)block * kKv4Block + (uint32_t)at, last = (uint32_t)end - 1;",
                            "const int32_t token = block * kKv4Block + at, last = end - 1;")
    assert signed != header
    run = places_check(tmp_path, signed)
    assert run.returncode == 1 and "differ" in run.stdout


# --------------------------------------------------------------- the reference

def test_reference_quantizer_properties():
    """At most half a step off inside the span, one at its ends; zero exact; s within 1/64 of the span's fifteenth."""
    g = np.random.default_rng(1)
    x = (g.standard_normal((400, 64)) * np.exp(g.uniform(-12, 9, (400, 1)))).astype(np.float32)
    x[5], x[6, :32] = 0, np.abs(x[6, :32])
    x[7, 3] = 0
    codes, words = ref.quantize(x)
    s = (words & 0xFFF0).view(np.float16).astype(np.float64)
    got = ref.value(codes, words)
    groups = x.reshape(400, 2, 32).astype(np.float64)
    span = np.maximum(groups.max(-1), 0) - np.minimum(groups.min(-1), 0)
    assert (15 * s >= span * (1 - 2.0 ** -23)).all()
    assert (s <= span / 15 * (1 + 2.0 ** -6) * (1 + 2.0 ** -22) + 2.0 ** -20).all()
    err = np.abs(got - x).reshape(400, 2, 32)
    assert (err <= 1.0 * s[..., None] + 1e-30).all()
    assert np.mean(err <= 0.5 * s[..., None] + 1e-30) > 0.95
    assert got[7, 3] == 0 and not got[5].any()
    assert (got.astype(np.float16) == got).all()


def test_reference_pages_return_what_was_put():
    g = np.random.default_rng(2)
    for page, dim in ((16, 64), (32, 128), (64, 256)):
        pages = ref.Pages(np.zeros((2, 3, page * (dim + dim // 8)), np.uint8), page, dim)
        kv = g.standard_normal((page, 2, 3, dim))
        for p in range(page):
            pages.put(1, p, *kv[p].astype(np.float32))
        for p in range(page):
            for got, x in zip(pages.get(1, p), kv[p]):
                assert np.array_equal(got, ref.value(*ref.quantize(x.astype(np.float32))))
        assert not pages.raw[0].any()


@pytest.mark.parametrize("change,message", [
    ({"heads": 0}, "heads must be"), ({"heads": 3}, "heads must be"), ({"window": -1}, "window"),
    ({"q_proj": (32, 128)}, "q_proj must have out_features 256"), ({"k_proj": (32, 256)}, "k_proj must have out_features 128"),
    ({"v_proj": (32, 256)}, "v_proj must have out_features 128"), ({"o_proj": (128, 32)}, "o_proj must have in_features 256"),
])
def test_attention_block_refusals(change, message):
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device="cpu")
    sizes = {"q_proj": (32, 256), "k_proj": (32, 128), "v_proj": (32, 128), "o_proj": (256, 32), **change}
    projections = {n: torch.nn.Linear(*sizes[n]) for n in ("q_proj", "k_proj", "v_proj", "o_proj")}
    options = {"heads": 4, **{n: v for n, v in change.items() if n in ("heads", "window")}}
    with pytest.raises(ValueError, match=message):
        AttentionBlock(**projections, cache=cache, **options)


def test_attention_block_refuses_inputs_that_need_gradients():
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device="cpu")
    block = AttentionBlock(torch.nn.Linear(32, 256), torch.nn.Linear(32, 128), torch.nn.Linear(32, 128),
                           torch.nn.Linear(256, 32), cache, heads=4)
    batch = PagedBatch(i32(2, 2), i32(2))
    x = torch.zeros(2, 32, requires_grad=True)
    with pytest.raises(ValueError, match="attn_input needs gradients"):
        block(x, x, batch)
    with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm GPU"):
        block(x, x, batch)


def test_attention_block_checks_its_rows():
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device="cpu")
    block = AttentionBlock(torch.nn.Linear(32, 256), torch.nn.Linear(32, 128), torch.nn.Linear(32, 128),
                           torch.nn.Linear(256, 32), cache, heads=4)
    batch = PagedBatch(i32(2, 2), i32(2))
    for x, residual in ((torch.zeros(2, 32), torch.zeros(2, 16)), (torch.zeros(3, 32), torch.zeros(3, 32)),
                        (torch.zeros(2, 1, 32), torch.zeros(2, 1, 32))):
        with pytest.raises(ValueError, match="attn_input and residual"):
            block(x, residual, batch)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        block(torch.zeros(2, 32), torch.zeros(2, 32), batch)
