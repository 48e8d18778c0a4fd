"""GPU parity of the 4-bit paged cache -- append with rotation, read, attention
-- with the 64-bit reference of kv4_reference.py: page bytes exactly,
attention within bounds derived from its roundings."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_reference as ref
from conftest import print_case
from drama_moe import _lib
from drama_moe.attention import KvCache4, PagedBatch, Rotary

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}
BAD = _lib.STATUS_BAD_BATCH


def wide(t):
    return t.detach().double().cpu().numpy()


class Case:
    """Sequences (new rows, tokens with them) over shuffled pages that first hold only `fill` bytes."""

    def __init__(self, cuda, seqs, hq, hkv, dim, page, dtype, *, seed=0, fill=0xFF, behind=0, spare=2, cols=None):
        g = torch.Generator().manual_seed(seed)
        self.g, self.cuda, self.seqs, self.dtype = g, cuda, seqs, dtype
        self.hq, self.hkv, self.dim, self.page = hq, hkv, dim, page
        need = [max(1, -(-length // page)) for _, length in seqs]
        count = sum(need) + spare
        order = torch.randperm(count, generator=g).int()
        self.table = torch.full((len(seqs), cols or max(need)), -7, dtype=torch.int32)
        at = 0
        for s, k in enumerate(need):
            self.table[s, :k] = order[at:at + k]
            at += k
        self.unused = order[at:].tolist()
        self.lengths = torch.tensor([length for _, length in seqs], dtype=torch.int32)
        self.starts = torch.tensor([0] + [n for n, _ in seqs], dtype=torch.int32).cumsum(0).int()
        self.rows = int(self.starts[-1]) + behind
        self.raw = torch.full((count, hkv, KvCache4.head_bytes(page, dim)), fill, dtype=torch.uint8)

    def random(self, heads, rows=None, std=1.0):
        return (torch.randn(self.rows if rows is None else rows, heads, self.dim, generator=self.g) * std).to(self.dtype)

    def fill(self):
        """Values at every place of every sequence, put there by the reference."""
        pages = ref.Pages(self.raw.numpy(), self.page, self.dim)
        for s, (_, length) in enumerate(self.seqs):
            kv = wide(torch.randn(length, 2, self.hkv, self.dim, generator=self.g) * 1.5)
            for p in range(length):
                pages.put(int(self.table[s, p // self.page]), p % self.page, *kv[p].astype(np.float32))
        return self

    def device(self, max_rows=None):
        cache = KvCache4(self.raw.to(self.cuda), page_size=self.page, head_dim=self.dim)
        batch = PagedBatch(self.table.to(self.cuda), self.lengths.to(self.cuda), self.starts.to(self.cuda),
                           rows=self.rows, max_rows=max_rows or max(1, max(n for n, _ in self.seqs)))
        return cache, batch

    def expected(self, q, scale, window=0):
        """(out, bound) over the rows that sequences own."""
        out, bound = np.zeros((self.rows, self.hq, self.dim)), np.zeros((self.rows, self.hq, self.dim))
        pages = ref.Pages(self.raw.numpy(), self.page, self.dim)
        for s, (n, length) in enumerate(self.seqs):
            if not n:
                continue
            k, v = pages.tokens(self.table[s].tolist(), length)
            at = slice(int(self.starts[s]), int(self.starts[s]) + n)
            o, size, terms = ref.attention(wide(q[at]), k, v, length, scale, window)
            out[at], bound[at] = o, ref.tolerance(o, size, terms, self.dim, max(length, 1), EPS[self.dtype])
        return out, bound


def check_attend(case, q, *, scale=None, window=0, status=0, max_rows=None):
    cache, batch = case.device(max_rows)
    scale = case.dim ** -0.5 if scale is None else scale
    want, bound = case.expected(q, scale, window)
    cache.status()
    out = torch.full((case.rows, case.hq, case.dim), 77.0, dtype=case.dtype, device=case.cuda)
    got = cache.attend(q.to(case.cuda), batch, scale=scale, window=window, out=out)
    assert got is out and cache.status() == status
    owned = int(case.starts[-1])
    over = np.abs(wide(out[:owned]) - want[:owned]) / bound[:owned]
    assert np.isfinite(over).all() and over.max() <= 1.0, over.max()
    assert (out[owned:] == 77.0).all()  # rows behind the last sequence
    again = cache.attend(q.to(case.cuda), batch, scale=scale, window=window)
    assert torch.equal(again[:owned], out[:owned])
    return out


# ------------------------------------------------------------- append and read

@pytest.mark.parametrize("dim,hq,hkv,page,dtype", [
    (64, 3, 3, 16, torch.float16), (64, 7, 1, 256, torch.bfloat16), (128, 8, 2, 32, torch.bfloat16),
    (128, 5, 5, 64, torch.float16), (256, 2, 1, 16, torch.bfloat16), (256, 4, 2, 128, torch.float16)])
@pytest.mark.parametrize("rot,interleaved,axes", [(1.0, False, 1), (0.5, False, 3), (0.25, True, 3), (1.0, True, 1)])
def test_append_writes_the_reference_bytes_and_nothing_else(cuda, dim, hq, hkv, page, dtype, rot, interleaved, axes):
    print_case("kv4 append", dim, hq, hkv, page, dtype, rot, interleaved, axes)
    seqs = [(1, 1), (5, 70), (0, 9), (16, 16), (33, page + 50), (3, 2), (2, 0)]  # the last two: rows without a place
    case = Case(cuda, seqs, hq, hkv, dim, page, dtype, seed=dim + axes, fill=0xA5, behind=3)
    qkv = case.random(hq + 2 * hkv)
    qkv[2, hq] = 0          # a key of zeros
    qkv[3, hq] *= 2.0 ** -14  # scales that are fp16 subnormals
    qkv[4, hq:] *= 300.0
    qkv[5, hq + hkv] = qkv[5, hq + hkv].abs() + 3  # no negative value
    half = int(dim * rot) // 2
    inv_freq = (10000.0 ** (-np.arange(half) / half)).astype(np.float32)
    axis = np.arange(half, dtype=np.uint8) % axes if axes > 1 else None
    positions = torch.randint(-20, 200000, (axes, case.rows), generator=case.g)
    cache, batch = case.device()
    rotary = Rotary(torch.from_numpy(inv_freq).to(cuda), axis=None if axis is None else torch.from_numpy(axis).to(cuda),
                    interleaved=interleaved)
    dev = qkv.to(cuda)
    q_out = torch.full((case.rows, hq, dim), 55.0, dtype=dtype, device=cuda)
    cache.status()
    got = cache.append(dev[:, hq:hq + hkv], dev[:, hq + hkv:], batch, rotary=rotary, q=dev[:, :hq], q_out=q_out,
                       positions=positions.to(cuda) if axes > 1 else positions[0].int().to(cuda))
    assert got is q_out and cache.status() == 0
    x = wide(qkv)
    turned = ref.rotate(x[:, :hq + hkv], positions.numpy(), inv_freq, axis, interleaved)
    pages = ref.Pages(case.raw.numpy(), page, dim)
    placed, held_k, held_v = [], [], []
    for s, (n, length) in enumerate(seqs):
        for i in range(n):
            row, p = int(case.starts[s]) + i, length - n + i
            if p < 0:
                continue
            at = (int(case.table[s, p // page]), p % page)
            pages.put(*at, turned[row, hq:].astype(np.float32), x[row, hq + hkv:])
            k, v = pages.get(*at)
            placed.append(row), held_k.append(k), held_v.append(v)
    assert np.array_equal(cache.pages.cpu().numpy(), pages.raw)
    assert len(placed) == 1 + 5 + 16 + 33 + 2
    # cosine and sine, a product and a sum rounded to fp32 (2^-24 each, of at most |a| + |b| <= sqrt(2) times the
    # pair's length, which is at most sqrt(2) times the head's largest value), then the result to the type
    err = np.abs(wide(q_out)[placed] - turned[placed, :hq])
    most = np.abs(x[placed, :hq]).max(-1, keepdims=True)
    assert (err <= EPS[dtype] / 2 * np.abs(turned[placed, :hq]) + 4 * 2.0 ** -24 * 2 * most * (1 + EPS[dtype]) + 2.0 ** -25).all()
    missing = sorted(set(range(case.rows)) - set(placed))
    assert (q_out[missing] == 55.0).all()
    k, v = cache.read(batch)
    assert k.dtype == torch.float16
    assert np.array_equal(wide(k)[placed], np.array(held_k)) and np.array_equal(wide(v)[placed], np.array(held_v))
    k16 = torch.full_like(k, 9.0, dtype=torch.bfloat16)
    v16 = torch.full_like(k16, 9.0)
    cache.read(batch, dtype=torch.bfloat16, k_out=k16, v_out=v16)
    assert torch.equal(k16[placed], k[placed].bfloat16()) and torch.equal(v16[placed], v[placed].bfloat16())
    assert (k16[missing] == 9.0).all() and (v16[missing] == 9.0).all()


def test_append_without_rotation_or_queries_and_in_place(cuda):
    print_case("kv4 append plain")
    case = Case(cuda, [(40, 100), (1, 1)], 4, 2, 128, 32, torch.bfloat16, seed=3, fill=0)
    cache, batch = case.device()
    k, v, q = case.random(2).to(cuda), case.random(2).to(cuda), case.random(4).to(cuda)
    assert cache.append(k, v, batch) is None
    plain = cache.pages.clone()
    # the own places as positions, in place, heads before rows in memory
    rotary = Rotary((10000.0 ** (-torch.arange(64) / 64)).to(cuda))
    places = torch.cat([torch.arange(60, 100), torch.tensor([0])]).to(cuda)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    a = cache.append(k, v, batch, rotary=rotary, positions=places, q=q)
    given = cache.pages.clone()
    b = cache.append(k, v, batch, rotary=rotary, q=swapped, q_out=swapped)
    assert b is swapped and torch.equal(a, b) and torch.equal(given, cache.pages)
    assert not torch.equal(plain, given)
    # channels in another order, rows at an odd address: copies of the inputs give the same
    odd = torch.empty(k.numel() + 1, dtype=k.dtype, device=cuda)[1:].view_as(k).copy_(k)
    turned = v.transpose(1, 2).contiguous().transpose(1, 2)
    cache.pages.zero_()
    cache.append(odd, turned, batch, rotary=rotary)
    assert torch.equal(given, cache.pages)
    # one head's rows broadcast to all
    cache.append(k[:1].expand(41, 2, 128), v, batch)
    assert torch.equal(cache.read(batch)[0][0], cache.read(batch)[0][40])


def test_values_no_code_can_stand_for(cuda):
    print_case("kv4 append non-finite")
    case = Case(cuda, [(4, 4)], 1, 1, 64, 16, torch.bfloat16, fill=0)
    k, v = case.random(1), case.random(1)
    k[1, 0, 3], k[2, 0, 5], v[1, 0, 40], v[3, 0, 7] = float("nan"), float("inf"), -1e30, float("-inf")
    cache, batch = case.device()
    cache.status()
    cache.append(k.to(cuda), v.to(cuda), batch)
    assert cache.status() == _lib.STATUS_NON_FINITE
    pages = ref.Pages(case.raw.numpy(), 16, 64)
    for i in range(4):
        pages.put(int(case.table[0, 0]), i, wide(k)[i], wide(v)[i])
    assert np.array_equal(cache.pages.cpu().numpy(), pages.raw)
    k, v = cache.read(batch)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    # the span is 32640 and a little from the other sign: the scale is the seven-bit number after 2176
    assert k[1, 0, 3] == 0 and k[2, 0, 5] == 15 * 2208 and v[1, 0, 40] == -15 * 2208


def test_ranges_at_and_beside_every_scale(cuda):
    """Groups whose range is 15 times a number of the scales' grid, exactly or the next fp16 value up or down."""
    print_case("kv4 scale grid")
    grid = [m * 2.0 ** (k - 6) for k in range(-14, 11) for m in range(64, 128)] + [m * 2.0 ** -20 for m in range(1, 64)]
    ranges = (15 * torch.tensor(grid, dtype=torch.float64)).half()
    assert (ranges.double() == 15 * torch.tensor(grid, dtype=torch.float64))[:64 * 25].all()
    bits = ranges.view(torch.int16)
    tops = torch.cat([ranges, (bits + 1).view(torch.float16), (bits - 1).view(torch.float16)])
    assert torch.isfinite(tops).all()
    heads, dim = 8, 64
    rows = -(-len(tops) // (heads * 2))
    k = torch.zeros(rows * heads * 2, 32, dtype=torch.float16)
    k[:len(tops), 5] = tops                    # all above zero
    v = torch.zeros_like(k)
    v[:len(tops), 9] = -tops                   # all below
    middle = torch.rand(k.shape, generator=torch.Generator().manual_seed(1)) * tops.max()
    k[:, 16:] = torch.minimum(middle[:, 16:].half(), k[:, 5:6])
    v[:, 16:] = -torch.minimum(middle[:, 16:].half() * 0.01, -v[:, 9:10])
    k, v = k.reshape(rows, heads, dim), v.reshape(rows, heads, dim)
    case = Case(cuda, [(rows, rows)], heads, heads, dim, 16, torch.float16, seed=2)
    cache, batch = case.device()
    cache.append(k.to(cuda), v.to(cuda), batch)
    pages = ref.Pages(case.raw.numpy(), 16, dim)
    for p in range(rows):
        pages.put(int(case.table[0, p // 16]), p % 16, wide(k)[p].astype(np.float32), wide(v)[p])
    assert np.array_equal(cache.pages.cpu().numpy(), pages.raw)


@pytest.mark.parametrize("dim,hq,hkv,rot,interleaved,dtype", [
    (128, 60, 2, 1.0, False, torch.bfloat16), (128, 80, 3, 0.5, True, torch.float16), (64, 50, 20, 1.0, False, torch.bfloat16),
    (256, 33, 16, 0.25, False, torch.float16)])
def test_a_large_call_is_its_small_ones(cuda, dim, hq, hkv, rot, interleaved, dtype):
    """Thousands of rows in one call against the same rows, up to 400 of one sequence a call."""
    print_case("kv4 large append", dim, hq, hkv, rot, interleaved, dtype)
    seqs = [(2000, 2000), (3, 700), (0, 5), (1337, 1400), (65, 65)]
    case = Case(cuda, seqs, hq, hkv, dim, 32, dtype, seed=hq, behind=7, fill=0)
    qkv = case.random(hq + 2 * hkv).to(cuda)
    half = int(dim * rot) // 2
    rotary = Rotary((10000.0 ** (-torch.arange(half) / half)).to(cuda), axis=Rotary.sections([half - 3, 2, 1], device=cuda),
                    interleaved=interleaved)
    positions = torch.randint(0, 90000, (3, case.rows), generator=case.g).to(cuda)
    cache, batch = case.device()
    cut = lambda at: (qkv[at, hq:hq + hkv], qkv[at, hq + hkv:])  # noqa: E731
    q_out = torch.full((case.rows, hq, dim), 3.0, dtype=dtype, device=cuda)
    cache.append(*cut(slice(None)), batch, rotary=rotary, positions=positions, q=qkv[:, :hq], q_out=q_out)
    k, v = (torch.full((case.rows, hkv, dim), 4.0, dtype=dtype, device=cuda) for _ in range(2))
    cache.read(batch, dtype=dtype, k_out=k, v_out=v)
    assert cache.status() == 0 and (q_out[-7:] == 3.0).all() and (k[-7:] == 4.0).all() and (v[-7:] == 4.0).all()
    pages = cache.pages.clone()
    cache.pages.zero_()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    for s, (n, length) in enumerate(seqs):
        for first in range(0, n, 400):
            count = min(400, n - first)
            at = slice(int(case.starts[s]) + first, int(case.starts[s]) + first + count)
            part = PagedBatch(batch.block_table[s:s + 1], i32(length - n + first + count), i32(0, count), rows=count)
            got = cache.append(*cut(at), part, rotary=rotary, positions=positions[:, at].contiguous(), q=qkv[at, :hq])
            assert torch.equal(got, q_out[at])
            kk, vv = cache.read(part, dtype=dtype)
            assert torch.equal(kk, k[at]) and torch.equal(vv, v[at])
    assert torch.equal(cache.pages, pages)


# ------------------------------------------------------------------- attention

EDGES = [(1, 1), (1, 2), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 128), (1, 300), (1, 1100)]


@pytest.mark.parametrize("dim,hq,hkv,page,dtype", [
    (64, 4, 4, 16, torch.float16), (64, 14, 2, 64, torch.bfloat16), (128, 16, 2, 16, torch.bfloat16),
    (128, 20, 1, 128, torch.float16), (128, 3, 1, 32, torch.bfloat16), (256, 8, 1, 256, torch.bfloat16),
    (256, 40, 1, 16, torch.float16)])
@pytest.mark.parametrize("window", [0, 70])
def test_one_token_a_sequence(cuda, dim, hq, hkv, page, dtype, window):
    print_case("kv4 decode", dim, hq, hkv, page, dtype, window)
    case = Case(cuda, EDGES, hq, hkv, dim, page, dtype, seed=dim + hq, behind=2).fill()
    check_attend(case, case.random(hq, std=1.5), window=window)


@pytest.mark.parametrize("dim,hq,hkv,page,dtype", [
    (64, 6, 2, 32, torch.bfloat16), (64, 5, 1, 16, torch.float16), (128, 8, 1, 64, torch.bfloat16),
    (128, 4, 4, 16, torch.float16), (128, 14, 2, 256, torch.bfloat16), (256, 4, 2, 64, torch.float16),
    (256, 3, 3, 16, torch.bfloat16)])
@pytest.mark.parametrize("seqs", [
    [(2, 2), (5, 80), (1, 40), (0, 30), (8, 8), (3, 129)],       # a few rows each, one sequence without
    [(17, 17), (64, 64), (65, 200), (1, 1), (130, 131)],         # prompts and chunks of odd lengths
    [(300, 411)],                                                # one chunk
    [(4, 2), (1, 0), (3, 3), (70, 66)],                          # rows before the first token see nothing
])
@pytest.mark.parametrize("window", [0, 33])
def test_several_rows_a_sequence(cuda, dim, hq, hkv, page, dtype, seqs, window):
    print_case("kv4 rows", dim, hq, hkv, page, dtype, seqs, window)
    case = Case(cuda, seqs, hq, hkv, dim, page, dtype, seed=dim + hq + len(seqs), behind=1).fill()
    out = check_attend(case, case.random(hq), window=window)
    for s, (n, length) in enumerate(seqs):
        empty = max(0, n - length)
        at = int(case.starts[s])
        assert (out[at:at + empty] == 0).all()


@pytest.mark.parametrize("dim,hq,hkv,seqs,longest,rows", [
    (64, 8, 4, 1300, 60, 1), (64, 2, 2, 1400, 190, 1), (128, 16, 8, 333, 64, 1), (256, 4, 2, 1100, 100, 1),
    (64, 5, 5, 900, 128, 1), (64, 8, 2, 700, 200, 6), (128, 12, 1, 600, 700, 2), (256, 8, 2, 300, 120, 9)])
@pytest.mark.parametrize("window", [0, 40])
def test_more_sequences_than_there_is_room_for(cuda, dim, hq, hkv, seqs, longest, rows, window):
    # several short sequences come to one wave or workgroup where they may be cut, and have their own where not
    print_case("kv4 crowd", dim, hq, hkv, seqs, longest, rows, window)
    lengths = torch.randint(1, longest + 1, (seqs,), generator=torch.Generator().manual_seed(seqs)).tolist()
    case = Case(cuda, [(min(n % 11, rows, n), n) for n in lengths], hq, hkv, dim, 64, torch.bfloat16, seed=seqs)
    # any codes, scales of 2^-7 to 2^-6 with any zero point
    case.raw.copy_(torch.randint(0, 256, case.raw.shape, dtype=torch.uint8, generator=case.g))
    scales = case.raw[:, :, 64 * dim:].view(torch.int16)
    scales.copy_(scales & 0x03FF | 0x2000)
    check_attend(case, case.random(hq), window=window)


@pytest.mark.parametrize("dim,group,rows", [
    (128, 1, 16), (128, 1, 17), (64, 8, 2), (64, 8, 3), (256, 1, 64), (256, 1, 65), (128, 32, 2), (128, 13, 5),
    (64, 1, 256), (64, 1, 257), (128, 8, 32), (128, 8, 33), (256, 2, 64), (256, 2, 65), (64, 128, 1), (128, 300, 1)])
def test_rows_at_the_edges_of_a_tile(cuda, dim, group, rows):
    print_case("kv4 tile edges", dim, group, rows)
    case = Case(cuda, [(rows, 1200), (rows, rows), (max(1, rows // 2), 65)], group, 1, dim, 32, torch.float16,
                seed=dim + group + rows).fill()
    q = case.random(group)
    q[0] *= 200.0  # scores that leave fp16 as weights of the base before
    check_attend(case, q, scale=dim ** -0.5)


def test_default_tables_and_strided_queries(cuda):
    """No starts: a row a sequence; q as a slice, heads first in memory, a broadcast row, an odd address."""
    print_case("kv4 attend strides")
    case = Case(cuda, [(1, 50), (1, 90), (1, 7)], 4, 2, 128, 16, torch.bfloat16, seed=5).fill()
    cache, _ = case.device()
    batch = PagedBatch(case.table.to(cuda), case.lengths.to(cuda))
    qkv = case.random(8).to(cuda)
    q = qkv[:, :4]
    want = cache.attend(q.contiguous(), batch)
    assert torch.equal(cache.attend(q, batch), want)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(cache.attend(heads_first, batch), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=cuda)[1:].view(q.shape).copy_(q)
    assert torch.equal(cache.attend(odd, batch), want)
    holder = torch.zeros(4, 3, 256, dtype=q.dtype, device=cuda)
    out = holder.transpose(0, 1)[:, :, 128:]
    assert torch.equal(cache.attend(q, batch, out=out), want)
    assert (holder[:, :, :128] == 0).all() and torch.equal(holder[:, :, 128:].transpose(0, 1), want)
    one = q[:1].expand(3, 4, 128)
    assert torch.equal(cache.attend(one, batch), cache.attend(one.contiguous(), batch))
    # table wider than needed, its rows strided
    table = torch.full((3, 40), -1, dtype=torch.int32, device=cuda)
    table[:, 5:5 + case.table.shape[1]] = case.table.to(cuda)
    assert torch.equal(cache.attend(q, PagedBatch(table[:, 5:30], batch.lengths)), want)


@pytest.mark.parametrize("rows", [1, 6, 150])
def test_odd_queries(cuda, rows):
    """Zero, tiny, huge and non-finite queries; a row that is no number stays alone with it."""
    print_case("kv4 odd queries", rows)
    case = Case(cuda, [(rows, 200)], 8, 2, 128, 32, torch.bfloat16, seed=6).fill()
    q = case.random(8)
    q[0, 0] = 0
    q[0, 1] *= 2.0 ** -100
    q[0, 2, :] = 0
    q[0, 2, 5] = 1e4  # one channel alone
    check_attend(case, q)
    clean = q.clone()
    cache, batch = case.device()
    q[0, 3, 7] = float("nan")
    q[0, 4, 9] = float("inf")
    got, want = cache.attend(q.to(cuda), batch), cache.attend(clean.to(cuda), batch)
    assert not torch.isfinite(got[0, 3:5]).any()
    got[0, 3:5] = want[0, 3:5]
    assert torch.equal(got, want)
    q = clean * 1e30  # scores far beyond exp's range: the largest alone counts
    out = cache.attend(q.to(cuda), batch)
    assert torch.isfinite(out[:, 3:]).all()


@pytest.mark.parametrize("dim,rows,length", [(64, 1, 40), (128, 1, 900), (256, 6, 1300), (64, 40, 300), (128, 40, 2000),
                                             (256, 20, 900), (128, 150, 200), (64, 300, 2500), (256, 140, 1200)])
def test_infinite_queries_whose_scores_are_all_negative(cuda, dim, rows, length):
    """A query with an infinity is no number in its result, also where every score is minus infinity; a row that sees
    no token is zero all the same."""
    print_case("kv4 infinite queries", dim, rows, length)
    case = Case(cuda, [(rows, length), (3, 1)], 4, 2, dim, 64, torch.bfloat16, seed=dim + rows, fill=0)
    cache, batch = case.device()
    for s, count in enumerate((length, 1)):
        k, v = (torch.randn(count, 2, dim, generator=case.g).to(cuda).bfloat16() for _ in range(2))
        k[:, :, 5] = -2.0
        cache.append(k, v, PagedBatch(batch.block_table[s:s + 1], batch.lengths[s:s + 1],
                                      torch.tensor([0, count], dtype=torch.int32, device=cuda), rows=count))
    q = case.random(4).to(cuda)
    want = cache.attend(q, batch)
    odd = [(0, 1), (rows - 1, 3), (rows, 0), (rows + 2, 2)]  # the last two of the second sequence's: its first row sees nothing
    for row, head in odd:
        q[row, head, 5] = float("inf")
    got = cache.attend(q, batch)
    for row, head in odd:
        assert (got[row, head] == 0).all() if row == rows else torch.isnan(got[row, head]).all()
        got[row, head] = want[row, head]
    assert torch.equal(got, want)


def test_scores_far_apart_and_many_equal(cuda):
    """Maxima that come first, last and in the middle; equal scores everywhere."""
    print_case("kv4 score ranges")
    case = Case(cuda, [(1, 700), (1, 700), (130, 700)], 2, 1, 64, 16, torch.float16, seed=8).fill()
    q = case.random(2)
    check_attend(case, q, scale=3.0)
    check_attend(case, q, scale=1e-6)
    check_attend(case, q * 0)


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_out_of_range_and_odd_batches_are_flagged_and_skipped(cuda, rows):
    print_case("kv4 bad batch", rows)
    seqs = [(rows, 150), (rows, 100), (rows, 60)]
    case = Case(cuda, seqs, 4, 2, 128, 16, torch.bfloat16, seed=9, spare=4).fill()
    q = case.random(4)
    good = check_attend(case, q)
    pages = len(case.raw)
    case.table[0, 2], case.table[1, 0], case.table[2, 1] = pages, -1, 2 ** 31 - 1
    check_attend(case, q, status=BAD)  # the reference leaves those tokens out too
    cache, batch = case.device()
    before = cache.pages.clone()
    k, v = case.random(2).to(cuda), case.random(2).to(cuda)
    cache.status()
    cache.append(k, v, batch)
    held = cache.read(batch)
    assert (cache.status() == BAD) == (rows > 1)
    if rows > 1:  # sequence 2's rows 20..59: those on its page 1 are not stored and read as 0
        gone = [2 * rows + p - 20 for p in range(20, 32)]
        assert all((x[gone] == 0).all() for x in held)
        kept = [r for r in range(3 * rows) if r not in gone and not (rows <= r < 2 * rows)]
        assert all((x[kept].float().abs().sum(-1) > 0).all() for x in held)
    case.table[0, 2] = case.table[1, 0] = case.table[2, 1] = 0

    def skipped(which, **changed):
        lengths, starts = changed.get("lengths", case.lengths), changed.get("starts", case.starts)
        bad = PagedBatch(batch.block_table, lengths.to(cuda), starts.to(cuda), rows=batch.rows,
                         max_rows=changed.get("max_rows", batch.max_rows))
        cache.pages.copy_(before)
        cache.status()
        cache.append(k, v, bad)
        assert cache.status() == BAD
        out = torch.full_like(good, 77.0)
        cache.attend(q.to(cuda), bad, out=out)
        assert cache.status() == BAD
        for s in range(3):
            mine = out[s * rows:(s + 1) * rows]
            assert (mine == 77.0).all() if s in which else torch.isfinite(mine).all() and not (mine == 77.0).any(), s
        return out

    batch.block_table.copy_(torch.where((case.table < 0) | (case.table >= pages), 0, case.table))
    skipped([1], lengths=torch.tensor([150, 2 ** 31 - 1, 60], dtype=torch.int32))
    skipped([0], lengths=torch.tensor([-5, 100, 60], dtype=torch.int32))
    skipped([2], starts=torch.tensor([0, rows, 2 * rows, 3 * rows + 1], dtype=torch.int32))
    skipped([0], starts=torch.tensor([-1, rows, 2 * rows, 3 * rows], dtype=torch.int32))
    if rows > 1:
        cut = case.starts.clone()
        cut[1] -= 1  # sequence 1 has one row more than max_rows says
        out = torch.full_like(good, 77.0)
        cache.attend(q.to(cuda), PagedBatch(batch.block_table, batch.lengths, cut.to(cuda), rows=batch.rows,
                                            max_rows=rows), out=out)
        assert cache.status() == BAD
        assert (out[rows - 1:2 * rows] == 77.0).all() and not (out[2 * rows:] == 77.0).any()


@pytest.mark.parametrize("heads,count", [(2, 6), (60, 3000)])
@pytest.mark.parametrize("what", ["behind the buffers", "back", "too long without rows", "negative without rows"])
def test_odd_sequences_without_rows_are_flagged(cuda, heads, count, what):
    """A sequence that is out of range is flagged by every call, also where none of the buffers' rows is its."""
    print_case("kv4 odd sequences", heads, count, what)
    case = Case(cuda, [(count, count)], heads, 2, 64, 64, torch.bfloat16, seed=count, fill=0)
    cache, batch = case.device()
    q, k, v = (case.random(h).to(cuda) for h in (heads, 2, 2))
    cache.status()
    cache.append(k, v, batch)
    stored, held = cache.pages.clone(), cache.read(batch)
    assert cache.status() == 0
    starts, lengths = {"behind the buffers": ([0, count, count, count + 4], [count, 0, 4]),
                       "back": ([0, count, count, 1], [count, 0, 0]),
                       "too long without rows": ([0, count, count, count], [count, 0, 2 ** 30]),
                       "negative without rows": ([0, count, count, count], [count, -1, 0])}[what]
    table = case.table.to(cuda).expand(3, -1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    odd = PagedBatch(table, i32(lengths), i32(starts), rows=count)
    cache.pages.zero_()
    cache.append(k, v, odd, q=q)
    assert cache.status() == BAD
    k_out, v_out = cache.read(odd)
    assert cache.status() == BAD
    if what != "back":  # where offsets go back, rows may be left out
        assert torch.equal(cache.pages, stored) and torch.equal(k_out, held[0]) and torch.equal(v_out, held[1])
    cache.attend(q, odd)
    assert cache.status() == BAD


@pytest.mark.parametrize("rows", [1, 10, 40])
def test_offsets_that_go_back(cuda, rows):
    """Every second sequence ends before it starts and is skipped; the others, all alike, own the same rows."""
    print_case("kv4 offsets back", rows)
    case = Case(cuda, [(rows, 3000)], 8, 2, 64, 64, torch.bfloat16, seed=rows).fill()
    cache, batch = case.device()
    q = case.random(8).to(cuda)
    cache.status()
    want = cache.attend(q, batch)
    assert cache.status() == 0
    n = 40
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table = case.table.to(cuda).expand(2 * n - 1, -1).contiguous()
    back = PagedBatch(table, i32([3000] * (2 * n - 1)), i32([0, rows] * n), rows=rows, max_rows=rows)
    got = torch.full_like(want, 5.0)
    cache.attend(q, back, out=got)
    assert cache.status() == BAD
    # other cuts of the same tokens: two roundings of the result, of weights and of sums apart
    bound = case.expected(q.cpu(), 64 ** -0.5)[1]
    assert (np.abs(wide(got) - wide(want)) <= 2 * bound).all()
    with pytest.raises(ValueError, match="window must fit"):
        cache.attend(q, batch, window=2 ** 32 + 5)


def test_places_beyond_32_bits(cuda):
    """Pages behind 4 GiB of others; a row buffer whose rows lie far apart."""
    print_case("kv4 far pages")
    free, _ = torch.cuda.mem_get_info(cuda)
    need = KvCache4.head_bytes(256, 128) * 4
    count = (5 << 30) // need
    assert free > 12 << 30
    raw = torch.empty(count, 4, need // 4, dtype=torch.uint8, device=cuda)
    cache = KvCache4(raw, page_size=256, head_dim=128)
    table = torch.tensor([[count - 1, 0, count - 2]], dtype=torch.int32, device=cuda)
    small = KvCache4.allocate(3, 4, 128, page_size=256, device=cuda)
    near = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(11)
    k, v, q = (torch.randn(700, 4, 128, generator=g).bfloat16().to(cuda) for _ in range(3))
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([700], [0, 700]))
    results = []
    for c, t in ((cache, table), (small, near)):
        batch = PagedBatch(t, lengths, starts, rows=700)
        c.append(k, v, batch)
        results.append((*c.read(batch), c.attend(q, batch), c.attend(q[:1].contiguous(), PagedBatch(t, lengths))))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    del raw, cache
    far = torch.empty(3 << 30, dtype=torch.bfloat16, device=cuda)
    spread = far.as_strided((3, 4, 128), ((1 << 30) + 64, 128, 1))
    spread.copy_(q[:3])
    batch = PagedBatch(near.expand(3, 3).contiguous(), lengths.expand(3).contiguous())
    assert torch.equal(small.attend(spread, batch), small.attend(q[:3].contiguous(), batch))


def test_shared_prefix_pages_and_strided_layers(cuda):
    """Two sequences on the same pages; a layer's pages inside a buffer of several layers."""
    print_case("kv4 shared pages")
    case = Case(cuda, [(1, 100)], 4, 2, 64, 16, torch.float16, seed=12).fill()
    cache, batch = case.device()
    q = case.random(4, rows=1).to(cuda)
    want = cache.attend(q, batch)
    twice = PagedBatch(case.table.to(cuda).expand(2, -1).contiguous(), case.lengths.to(cuda).expand(2).contiguous())
    both = cache.attend(q.expand(2, 4, 64), twice)
    assert torch.equal(both[0], want[0]) and torch.equal(both[1], want[0])
    layers = torch.full((case.raw.shape[0], 3, *case.raw.shape[1:]), 0xFF, dtype=torch.uint8, device=cuda)
    layers[:, 1] = cache.pages
    inner = KvCache4(layers[:, 1], page_size=16, head_dim=64)
    assert torch.equal(inner.attend(q, batch), want)


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_one_table_row_for_all_sequences(cuda, rows):
    """A table expanded from one row is its copy: sequences on the same pages, each at places of its own."""
    print_case("kv4 expanded table", rows)
    case = Case(cuda, [(rows, 300)], 4, 2, 64, 16, torch.bfloat16, seed=rows + 50).fill()
    n = 5
    cache, _ = case.device()
    lengths = torch.tensor([300, 60, 107, 154, 201], dtype=torch.int32, device=cuda)
    starts = torch.arange(0, n * rows + 1, rows, dtype=torch.int32, device=cuda)
    q, k, v = (case.random(h, rows=n * rows).to(cuda) for h in (4, 2, 2))
    table = case.table.to(cuda)
    before, results = cache.pages.clone(), []
    cache.status()
    for t in (table.expand(n, -1), table.expand(n, -1).contiguous()):
        cache.pages.copy_(before)
        batch = PagedBatch(t, lengths, starts, rows=n * rows, max_rows=rows)
        first = cache.attend(q, batch)
        cache.append(k, v, batch)
        results.append((first, cache.pages.clone(), *cache.read(batch), cache.attend(q, batch, window=50)))
    assert cache.status() == 0 and not torch.equal(results[0][1], before)
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dim,hq,hkv", [(64, 2, 2), (128, 4, 1), (256, 1, 1)])
@pytest.mark.parametrize("rows", [1, 3, 20, 70])
def test_the_last_of_the_longest_sequence(cuda, dim, hq, hkv, rows):
    """2^31 - 1 tokens, of which a window sees the last: blocks and places at the end of 31 bits."""
    print_case("kv4 longest", dim, hq, hkv, rows)
    page, longest, window = 256, 2 ** 31 - 1, 300
    cols = -(-longest // page)
    table = torch.full((1, cols), 4, dtype=torch.int32, device=cuda)
    table[0, -4:] = torch.tensor([3, 0, 2, 1], dtype=torch.int32)
    cache = KvCache4.allocate(5, hkv, dim, page_size=page, device=cuda)
    base, n = (cols - 4) * page, 900
    g = torch.Generator().manual_seed(dim + rows)
    k, v = (torch.randn(n, hkv, dim, generator=g).half() for _ in range(2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    cache.status()
    cache.append(k.to(cuda), v.to(cuda), PagedBatch(table, i32(longest), i32(0, n), rows=n))
    pages = ref.Pages(np.zeros(cache.pages.shape, np.uint8), page, dim)
    own, places = [3, 0, 2, 1], range(longest - base - n, longest - base)
    for i, p in enumerate(places):
        pages.put(own[p // page], p % page, wide(k)[i], wide(v)[i])
    assert np.array_equal(cache.pages.cpu().numpy(), pages.raw)
    batch = PagedBatch(table, i32(longest), i32(0, rows), rows=rows)
    q = torch.randn(rows, hq, dim, generator=g).half()
    out = cache.attend(q.to(cuda), batch, window=window)
    held = [np.stack(x) for x in zip(*(pages.get(own[p // page], p % page) for p in range(longest - base)))]
    want, size, terms = ref.attention(wide(q), *held, longest - base, dim ** -0.5, window)
    bound = ref.tolerance(want, size, terms, dim, window, EPS[torch.float16])
    assert cache.status() == 0 and (np.abs(wide(out) - want) <= bound).all()
    got = cache.read(batch)
    assert all(np.array_equal(wide(x), y[-rows:]) for x, y in zip(got, held))


@pytest.mark.parametrize("dim,hq,hkv,page,window,rows", [
    (128, 16, 2, 16, 70, 1), (64, 4, 4, 32, 33, 1), (256, 2, 1, 16, 100, 3), (128, 4, 1, 32, 65, 12),
    (64, 10, 2, 16, 40, 9), (256, 8, 1, 16, 50, 5), (128, 2, 1, 16, 90, 150), (256, 3, 3, 32, 130, 130),
    (64, 4, 1, 16, 64, 200)])
def test_pages_behind_a_window_may_be_given_back(cuda, dim, hq, hkv, page, window, rows):
    """Table entries of which no row sees a token name no page: nothing is flagged.  The first one in sight is."""
    print_case("kv4 window pages", dim, hq, hkv, page, window, rows)
    lengths = [rows + x for x in (0, 257, 300, 313, 326, 350)]
    case = Case(cuda, [(rows, length) for length in lengths], hq, hkv, dim, page, torch.bfloat16, seed=dim + rows).fill()
    q = case.random(hq)
    gone = [max(0, length - rows - window + 1) // page for length in lengths]
    for s, count in enumerate(gone):
        case.table[s, :count] = torch.tensor([-1, len(case.raw), 2 ** 31 - 1, -2 ** 31]).repeat(99)[:count].int()
    assert gone[0] == 0 and min(gone[1:]) > 0
    check_attend(case, q, window=window)
    case.table[3, gone[3]] = -1
    check_attend(case, q, window=window, status=BAD)


@pytest.mark.parametrize("dim,hq,hkv,page,window,rows", [
    (128, 16, 2, 16, 70, 1), (64, 4, 4, 256, 33, 1), (256, 2, 1, 128, 100, 3), (128, 4, 1, 32, 65, 12),
    (64, 10, 2, 64, 40, 9), (256, 8, 1, 16, 50, 5), (128, 2, 1, 64, 90, 150), (256, 3, 3, 128, 130, 130),
    (64, 4, 1, 16, 64, 200)])
def test_slots_behind_a_window_may_hold_anything(cuda, dim, hq, hkv, page, window, rows):
    """Tokens that no row sees were never stored: their slots, and pages named in their place, hold bytes of 255 (scales
    that are no number)."""
    print_case("kv4 window slots", dim, hq, hkv, page, window, rows)
    lengths = [rows + x for x in (0, 257, 300, 313, 326, 350, 366)]
    case = Case(cuda, [(rows, length) for length in lengths], hq, hkv, dim, page, torch.bfloat16, seed=dim + page)
    clean = ref.Pages(case.raw.numpy().copy(), page, dim)
    pages = ref.Pages(case.raw.numpy(), page, dim)
    for s, length in enumerate(lengths):
        kv = wide(torch.randn(length, 2, hkv, dim, generator=case.g)).astype(np.float32)
        lowest = max(0, length - rows - window + 1)
        for p in range(length):
            at = (int(case.table[s, p // page]), p % page)
            clean.put(*at, *kv[p])
            if p >= lowest:
                pages.put(*at, *kv[p])
    q = case.random(hq)
    stored = case.raw.clone()
    case.raw = torch.from_numpy(clean.raw)
    want = check_attend(case, q, window=window)
    case.raw = stored
    for s, length in enumerate(lengths):
        case.table[s, :max(0, length - rows - window + 1) // page] = case.unused[s % 2]
    cache, batch = case.device()
    cache.status()
    got = cache.attend(q.to(cuda), batch, window=window)
    assert torch.isfinite(got).all() and torch.equal(got, want) and cache.status() == 0


@pytest.mark.parametrize("dim,hq,hkv,window", [(64, 4, 2, 0), (128, 8, 1, 0), (128, 2, 2, 1500), (256, 2, 1, 0)])
@pytest.mark.parametrize("order", ["long last", "long first", "many between"])
def test_cut_and_whole_tiles_in_one_batch(cuda, dim, hq, hkv, window, order):
    """Sequences of many rows: some end in one piece, some are cut, more than 64 of them."""
    print_case("kv4 mixed cuts", dim, hq, hkv, window, order)
    short, long = [(9, 9), (1, 70), (0, 12), (40, 41)], [(130, 2600), (3, 3000), (1, 1990)]
    seqs = {"long last": short + [(140, 150)] + long, "long first": long + short,
            "many between": long[:1] + short * 17 + long[1:] + short}[order]
    case = Case(cuda, seqs, hq, hkv, dim, 64, torch.bfloat16, seed=dim + hq + len(seqs), behind=2)
    case.raw.copy_(torch.randint(0, 256, case.raw.shape, dtype=torch.uint8, generator=case.g))
    scales = case.raw[:, :, 64 * dim:].view(torch.int16)
    scales.copy_(scales & 0x03FF | 0x2000)  # 2^-7 to 2^-6 with any zero point
    check_attend(case, case.random(hq), window=window)


# --------------------------------------------------------------- as it is used

def decode_step(cache, batch, qkv, hq, hkv, rotary):
    q = cache.append(qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], batch, rotary=rotary, q=qkv[:, :hq])
    return cache.attend(q, batch)


def test_prompt_in_one_call_in_chunks_and_token_by_token(cuda):
    """The same tokens appended at once, in chunks and singly leave the same pages; attention agrees."""
    print_case("kv4 prompt ways")
    hq, hkv, dim, n = 8, 2, 128, 150
    g = torch.Generator().manual_seed(21)
    qkv = torch.randn(n, hq + 2 * hkv, dim, generator=g).half().to(cuda)
    rotary = Rotary((10000.0 ** (-torch.arange(64) / 64)).to(cuda))
    table = torch.tensor([[4, 1, 3, 0, 2]], dtype=torch.int32, device=cuda)
    results = []
    for sizes in ([n], [64, 1, 7, 78], [1] * n):
        cache = KvCache4.allocate(5, hkv, dim, page_size=32, device=cuda)
        outs, at = [], 0
        for size in sizes:
            i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
            batch = PagedBatch(table, i32(at + size), i32(0, size), rows=size)
            outs.append(decode_step(cache, batch, qkv[at:at + size], hq, hkv, rotary))
            at += size
        results.append((cache.pages, torch.cat(outs)))
    for pages, out in results[1:]:
        assert torch.equal(pages, results[0][0])
        # both within the bound of the reference: weights' fp16 rounding, sums, the result's rounding, twice
        assert (out.float() - results[0][1].float()).abs().max() <= 2 * (2.0 ** -10 + 2.0 ** -11) * 6


@pytest.mark.parametrize("seqs,longest", [(3, 1), (2, 40)])
def test_captured_steps_replay_with_other_tables(cuda, seqs, longest):
    """Two graphs over one cache, captured apart and replayed in turn with eager calls between, as tables change."""
    print_case("kv4 graphs", seqs, longest)
    hq, hkv, dim, page = 8, 2, 128, 16
    g = torch.Generator().manual_seed(31)
    rotary = Rotary((10000.0 ** (-torch.arange(64) / 64)).to(cuda))
    cache = KvCache4.allocate(64, hkv, dim, page_size=page, device=cuda)
    rows = seqs * longest + 2
    table = torch.randperm(64, generator=g)[:seqs * 16].reshape(seqs, 16).int().to(cuda)
    lengths = torch.full((seqs,), longest, dtype=torch.int32, device=cuda)
    starts = torch.arange(0, seqs * longest + 1, longest, dtype=torch.int32, device=cuda)
    qkv = torch.randn(rows, hq + 2 * hkv, dim, generator=g).bfloat16().to(cuda)
    batch = PagedBatch(table, lengths, starts, rows=rows, max_rows=longest)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode_step(cache, batch, qkv, hq, hkv, rotary)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = decode_step(cache, batch, qkv, hq, hkv, rotary)
        graphs.append((graph, out))
    for step, length in enumerate([longest, 60, 61, 200, 256, longest, 130]):
        lengths.copy_(torch.tensor([max(longest, length - 17 * s) for s in range(seqs)], dtype=torch.int32))
        qkv.copy_(torch.randn(rows, hq + 2 * hkv, dim, generator=g).bfloat16())
        graph, out = graphs[step % 2]
        graph.replay()
        torch.cuda.synchronize()
        pages = cache.pages.clone()
        want = decode_step(cache, batch, qkv, hq, hkv, rotary)
        assert torch.equal(out[:seqs * longest], want[:seqs * longest]) and torch.equal(pages, cache.pages), step
    # a padded slot: a sequence of no tokens stores nothing and its rows become 0
    lengths[0] = 0
    before = cache.pages.clone()
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert (graphs[0][1][:longest] == 0).all()
    mine = table[0].long()
    assert torch.equal(cache.pages[mine], before[mine])
    assert cache.status() == 0


def test_calls_on_two_streams_at_once(cuda):
    print_case("kv4 streams")
    case = Case(cuda, [(1, 900), (1, 350)], 16, 2, 128, 16, torch.bfloat16, seed=41).fill()
    cache, batch = case.device()
    qs = [case.random(16).to(cuda) for _ in range(6)]
    want = [cache.attend(q, batch) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(cache.attend(q, batch))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_inputs_that_need_gradients_are_refused(cuda):
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device=cuda)
    batch = PagedBatch(*(torch.ones(s, dtype=torch.int32, device=cuda) for s in ((2, 2), (2,))))
    k, grad = (torch.ones(2, 2, 64, dtype=torch.bfloat16, device=cuda).requires_grad_(x) for x in (False, True))
    pages = cache.pages.clone()
    calls = [(lambda: cache.append(grad, k, batch), "k needs"), (lambda: cache.append(k, grad, batch), "v needs"),
             (lambda: cache.append(k, k, batch, q=grad), "q needs"), (lambda: cache.attend(grad, batch), "q needs"),
             (lambda: cache.append(k, k, batch, q=k, q_out=grad), "q_out needs"),
             (lambda: cache.attend(k, batch, out=grad), "out needs"),
             (lambda: cache.read(batch, dtype=torch.bfloat16, k_out=grad), "k_out needs")]
    for call, message in calls:
        with pytest.raises(ValueError, match=message + " gradients"):
            call()
    assert torch.equal(cache.pages, pages)
    want = cache.append(k, k, batch, q=k), cache.attend(k, batch)
    with torch.no_grad():
        got = cache.append(grad, grad, batch, q=grad), cache.attend(grad, batch)
    with torch.inference_mode():
        again = cache.append(grad, grad, batch, q=grad), cache.attend(grad, batch)
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c) and not b.requires_grad


def test_calls_that_are_refused(cuda):
    cache = KvCache4.allocate(4, 2, 64, page_size=16, device=cuda)
    batch = PagedBatch(*(torch.ones(s, dtype=torch.int32, device=cuda) for s in ((2, 2), (2,))))
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=cuda)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=cuda)
    rotary = Rotary(torch.ones(32, device=cuda))
    places = torch.zeros(2, dtype=torch.int64, device=cuda)
    pages = cache.pages.clone()
    for call, message in [
        (lambda: cache.append(k.float(), k, batch), "k must be bf16 or fp16"),
        (lambda: cache.append(k, k.half(), batch), "v must be"),
        (lambda: cache.append(k[:1], k, batch), r"k must be \[2, 2, 64\]"),
        (lambda: cache.append(k, k.cpu(), batch), "v must be on"),
        (lambda: cache.append(k, k, batch, q_out=q), "q_out needs q"),
        (lambda: cache.append(k, k, batch, q=q.half()), "q must be"),
        (lambda: cache.append(k, k, batch, q=q, q_out=q[:, :2]), "q_out must be"),
        (lambda: cache.append(k, k, batch, q=q, q_out=q.transpose(1, 2).contiguous().transpose(1, 2)), "16-byte"),
        (lambda: cache.append(k, k, batch, positions=places), "positions need a rotary"),
        (lambda: cache.append(k, k, batch, rotary=Rotary(torch.ones(40, device=cuda))), "more rotated channels"),
        (lambda: cache.append(k, k, batch, rotary=Rotary(torch.ones(32))), "share a device"),
        (lambda: cache.append(k, k, batch, rotary=rotary, positions=places.float()), "positions must be int32"),
        (lambda: cache.append(k, k, batch, rotary=rotary, positions=places[:1]), "positions must be"),
        (lambda: cache.append(k, k, batch, rotary=rotary, positions=places.cpu()), "positions must be on"),
        (lambda: cache.append(k, k, batch, rotary=rotary, positions=places[None][:0]), "no axis"),
        (lambda: cache.read(batch, dtype=torch.float32), "k_out must be bf16"),
        (lambda: cache.read(batch, k_out=k), "k_out must be"),
        (lambda: cache.attend(q[:, :3], batch), "multiple of the key/value heads"),
        (lambda: cache.attend(q.float(), batch), "q must be bf16 or fp16"),
        (lambda: cache.attend(q, batch, out=q.half()), "out must be"),
        (lambda: cache.attend(q, batch, scale=-1.0), "scale must be positive"),
        (lambda: cache.attend(q, batch, window=-3), "window must not"),
        (lambda: cache.attend(q, PagedBatch(i32 := torch.ones(2, 2, dtype=torch.int32), i32[0])), "share a device"),
    ]:
        with pytest.raises(ValueError, match=message):
            call()
    torch.cuda.synchronize()
    assert torch.equal(cache.pages, pages)
    # a call without rows does nothing
    none = PagedBatch(batch.block_table, batch.lengths, torch.zeros(3, dtype=torch.int32, device=cuda), rows=0)
    assert cache.append(k[:0], k[:0], none, q=q[:0]).shape == (0, 4, 64)
    assert cache.read(none)[0].shape == (0, 2, 64) and cache.attend(q[:0], none).shape == (0, 4, 64)
