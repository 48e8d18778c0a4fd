// How an attention call over the 4-bit cache is cut into workgroups.
//
// Lengths live on the device (a captured step is replayed with other ones), so
// the cut is made there: every wave reads the lengths and finds its
// workgroup's part.  A part of a tile's blocks that is not all of them leaves
// an unnormalised partial sum, which a second launch joins.
//
// Few rows a sequence (one tile each): the blocks of 64 tokens of all
// sequences and key/value heads, laid end to end, are dealt out in equal
// shares, so a long sequence among short ones is spread over the whole chip
// and every workgroup ends at the same time; a share may span the end of one
// sequence and the start of the next.  If the sequences fill whole shares
// without needing more workgroups than there are, shares end with them.
//
// Many rows: tiles of different length, each cut into pieces of at most the
// average work of a workgroup, the longest tiles of a sequence first.  Only
// the pieces of cut tiles have a place for a partial sum.
#pragma once

#include "common.hpp"
#include "kv4.hpp"

namespace dmoe {

// A workgroup's next piece of work: blocks [from, to) of a tile.
struct Kv4Segment {
    int seq, head, row0, n, len;
    int row_a;     // first packed row of the tile
    int from, to;
    bool whole;    // all blocks of the tile: the result is final
    int64_t slot;  // where its partial sum goes
};

// The wave's index in its workgroup and a lane's value, known to the compiler
// to be the same in all lanes: block counters, tables and branches stay scalar.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ __forceinline__ int of_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// The lane's index, as of the segment that it works on: what is computed from
// it is not kept in registers from one segment to the next.
__device__ __forceinline__ int segment_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // the row before's last lane, into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int wave_total(int v) { return of_lane(wave_scan(v), kWave - 1); }

// The first token that a row at place p sees; no row behind it sees an earlier one.
__device__ __forceinline__ int kv4_lowest(int p, int window) {
    return window > 0 ? (int)max((int64_t)0, (int64_t)p - window + 1) : 0;
}

// First and last (exclusive) block that rows i0..i1 of a sequence see.
__device__ __forceinline__ void kv4_blocks(const Kv4Seq& q, int window, int i0, int i1, int& b0, int& b1) {
    const int p0 = q.len - q.n + i0, p1 = q.len - q.n + i1;
    b0 = kv4_lowest(p0, window) / kKv4Block;
    b1 = p1 < 0 ? b0 : max(b0, p1 / kKv4Block + 1);
}

// 64 sequences of the batch, one a lane.
struct Kv4Lane {
    Kv4Seq q;
    int b0, blocks;  // blocks that any of its rows sees
};
__device__ __forceinline__ Kv4Lane kv4_lane(const Kv4AttendArgs& a, int s) {
    Kv4Lane l{{0, 0, 0}, 0, 0};
    if (s >= a.batch.seqs) return l;
    bool bad;
    l.q = kv4_seq(a.batch, a.cache.page_shift, s, bad);
    if (bad && blockIdx.x == 0 && a.status) raise_status(a.status, kBadBatch);
    if (l.q.n) {
        int b1;
        kv4_blocks(l.q, a.window, 0, l.q.n - 1, l.b0, b1);
        l.blocks = b1 - l.b0;
    }
    return l;
}

// What the join of a tile's partial sums needs to know of it.
struct alignas(16) Kv4Record {
    int pieces, first;  // partial sums, and the workgroup that has the first
    int row0, n;
};

// Equal shares of all blocks, one tile a sequence.
struct Kv4Shares {
    const Kv4AttendArgs& a;
    int index;  // of the workgroup, or of the wave where each has a share
    int share, x, x_end, s0;
    bool padded;
    Kv4Lane lane;
    int extent, upto;  // of this lane's sequence; with all before it

    // every sequence has a place, also one that sees nothing: its rows become zero
    __device__ __forceinline__ int fit(int blocks) const {
        return padded ? (max(blocks, 1) + share - 1) / share * share : max(blocks, 1);
    }
    __device__ __forceinline__ void place(int before) {
        const int s = s0 + (int)(threadIdx.x & 63);
        extent = s < a.batch.seqs ? fit(lane.blocks) : 0;
        upto = before + wave_scan(extent);
    }

    __device__ Kv4Shares(const Kv4AttendArgs& args, int index_) : a(args), index(index_), s0(0), padded(false) {
        const int seqs = a.batch.seqs, kv = a.cache.kv_heads, me = threadIdx.x & 63;
        const bool once = seqs <= kWave;
        int total = 0;
        for (int s = 0; s < seqs; s += kWave) {
            lane = kv4_lane(a, s + me);
            total += wave_total(s + me < seqs ? max(lane.blocks, 1) : 0);
        }
        const int slots = 1 << a.slots_log2;
        share = a.min_blocks;
        int shares = seqs;
        if (a.cut) {
            share = max(share, (int)(((int64_t)total * kv + slots - 1) >> a.slots_log2));
            shares = 0;
            for (int s = 0; s < seqs; s += kWave) {
                if (!once) lane = kv4_lane(a, s + me);
                shares += wave_total(s + me < seqs ? (max(lane.blocks, 1) + share - 1) / share : 0);
            }
        }
        // where nothing is cut a tile has a share to itself, however many there are
        padded = !a.cut || (int64_t)shares * kv <= slots;
        const int end = (padded ? shares * share : total) * kv;
        x = (int)min((int64_t)index * share, (int64_t)end);
        x_end = min(x + share, end);
        if (!once) lane = kv4_lane(a, me);
        place(0);
    }

    __device__ __forceinline__ bool next(Kv4Segment& g) {
        if (x >= x_end) return false;
        const int kv = a.cache.kv_heads;
        unsigned long long past;
        while (!(past = __ballot((int64_t)upto * kv > x))) {
            // lengths written over while the kernel runs can leave less than was counted: the wave ends all the same
            if (s0 + kWave >= a.batch.seqs) {
                x = x_end;
                return false;
            }
            const int before = of_lane(upto, kWave - 1);
            s0 += kWave;
            lane = kv4_lane(a, s0 + (int)(threadIdx.x & 63));
            place(before);
        }
        const int who = __ffsll(past) - 1;
        const int size = of_lane(extent, who), rel = x - (of_lane(upto, who) - size) * kv;
        const int blocks = of_lane(lane.blocks, who), b0 = of_lane(lane.b0, who);
        g.seq = s0 + who;
        g.head = rel / size;
        g.row0 = of_lane(lane.q.row0, who);
        g.n = of_lane(lane.q.n, who);
        g.len = of_lane(lane.q.len, who);
        g.row_a = 0;
        const int at = rel - g.head * size, more = min(size - at, x_end - x);
        g.from = b0 + min(at, blocks);
        g.to = b0 + min(at + more, blocks);
        // the tile's places in the row of shares; padding behind its blocks is no piece
        const int x0 = x - at, x1 = x0 + max(blocks, 1), first = x0 / share, pieces = (x1 - 1) / share - first + 1;
        g.whole = pieces == 1;
        g.slot = 2 * (int64_t)index + (at == 0);
        if (at == 0 && (threadIdx.x & 63) == 0 && a.records)
            a.records[(int64_t)g.seq * kv + g.head] = Kv4Record{g.n ? pieces : 0, first, g.row0, g.n};
        x += more;
        return true;
    }
};

// Tiles and pieces of them, one a workgroup.  kTiles: workgroup `index` of the
// pass over whole tiles that joins their pieces.
struct Kv4Item {
    int seq, head, tile, split, splits;
    int row0, n, len;
    int first;  // workgroup of the tile's first piece; its pieces lie kv_heads apart,
    int slot;   // as do their partial sums, which only cut tiles have
    bool live;
};

template <bool kTiles>
__device__ Kv4Item kv4_item(const Kv4AttendArgs& a, int index) {
    const int lane = threadIdx.x & 63, kv = a.cache.kv_heads, seqs = a.batch.seqs;
    const bool once = seqs <= kWave;
    Kv4Lane l;
    int tiles = 0;
    const auto load = [&](int s) {
        l = kv4_lane(a, s + lane);
        tiles = (int)(((int64_t)l.q.n * a.group + a.tile_rows - 1) / a.tile_rows);
    };
    int work = 0;
    for (int s = 0; s < seqs; s += kWave) {
        load(s);
        work += wave_total(tiles * l.blocks);
    }
    const int piece = max(a.min_blocks, (int)(((int64_t)work * kv + (1 << a.slots_log2) - 1) >> a.slots_log2));
    Kv4Item it;
    it.live = false;
    it.head = index % kv;
    const int want = index / kv;
    int before = 0, pieces_before = 0, slots_before = 0;
    for (int s = 0; s < seqs; s += kWave) {
        if (!once) load(s);
        const int splits = l.blocks <= kKv4Whole ? 1 : (l.blocks + piece - 1) / piece;
        const int mine = kTiles ? tiles : tiles * splits;
        const int cut = splits > 1 ? tiles * splits : 0;
        const int upto = wave_scan(mine), pieces = wave_scan(tiles * splits), slots = wave_scan(cut);
        const unsigned long long past = __ballot(before + upto > want);
        if (past) {
            const int who = __ffsll(past) - 1;
            it.seq = s + who;
            it.splits = of_lane(splits, who);
            it.row0 = of_lane(l.q.row0, who);
            it.n = of_lane(l.q.n, who);
            it.len = of_lane(l.q.len, who);
            const int at = want - (before + of_lane(upto - mine, who));
            const int first = pieces_before + of_lane(pieces - tiles * splits, who);
            it.tile = kTiles ? at : at / it.splits;
            it.split = kTiles ? 0 : at % it.splits;
            it.first = (first + it.tile * it.splits) * kv + it.head;
            it.slot = (slots_before + of_lane(slots - cut, who) + it.tile * it.splits) * kv + it.head;
            it.tile = of_lane(tiles, who) - 1 - it.tile;  // the last rows see the most
            it.live = true;
            return it;
        }
        before += of_lane(upto, kWave - 1);
        pieces_before += of_lane(pieces, kWave - 1);
        slots_before += of_lane(slots, kWave - 1);
    }
    return it;
}

// This workgroup's piece of a tile; false if there is none.
__device__ __forceinline__ bool kv4_piece(const Kv4AttendArgs& a, Kv4Segment& g) {
    const Kv4Item it = kv4_item<false>(a, blockIdx.x);
    if (!it.live) return false;
    g = Kv4Segment{it.seq, it.head, it.row0, it.n, it.len, it.tile * a.tile_rows, 0, 0, it.splits == 1, it.slot + (int64_t)it.split * a.cache.kv_heads};
    const int last = min(g.row_a + a.tile_rows, g.n * a.group) - 1;
    int b0, b1;
    kv4_blocks(Kv4Seq{g.row0, g.n, g.len}, a.window, g.row_a / a.group, last / a.group, b0, b1);
    const uint32_t each = (uint32_t)(b1 - b0) / (uint32_t)it.splits, more = (uint32_t)(b1 - b0) - each * it.splits;
    g.from = b0 + it.split * (int)each + min(it.split, (int)more);
    g.to = g.from + (int)each + (it.split < (int)more ? 1 : 0);
    return true;
}

}  // namespace dmoe
