// How an attention call over the 4-bit cache is cut into workgroups.
//
// Lengths live on the device (a captured step is replayed with other ones), so
// the cut is made there: every wave reads the lengths, adds up the blocks of
// 64 tokens that all tiles see, and from that takes the same piece size.  A
// tile of a sequence becomes as many pieces as its sequence's blocks hold that
// size; a long sequence among short ones is spread over the whole chip.
#pragma once

#include "common.hpp"
#include "kv4.hpp"

namespace dmoe {

struct Kv4Item {
    int seq, head, tile, split, splits;
    int row0, n, len;
    int first;  // workgroup index of the tile's first piece, its pieces lie kv_heads apart
    bool live;
};

// The wave's index in its workgroup and a lane's value, known to the compiler
// to be the same in all lanes: block counters, tables and branches stay scalar.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ __forceinline__ int of_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

__device__ __forceinline__ int64_t wave_sum_i64(int64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// First and last (exclusive) block that rows i0..i1 of a sequence see.
__device__ __forceinline__ void kv4_blocks(const Kv4Seq& q, int window, int i0, int i1, int& b0, int& b1) {
    const int p0 = q.len - q.n + i0, p1 = q.len - q.n + i1;
    b0 = window > 0 ? max(0, (int)max((int64_t)0, (int64_t)p0 - window + 1)) / kKv4Block : 0;
    b1 = p1 < 0 ? b0 : max(b0, p1 / kKv4Block + 1);
}

// The blocks [from, to) of a piece of a tile that sees blocks [b0, b1).
__device__ __forceinline__ void kv4_piece(const Kv4Item& it, int b0, int b1, int& from, int& to) {
    const uint32_t each = (uint32_t)(b1 - b0) / (uint32_t)it.splits, more = (uint32_t)(b1 - b0) - each * it.splits;
    from = b0 + it.split * (int)each + min(it.split, (int)more);
    to = from + (int)each + (it.split < (int)more ? 1 : 0);
}

// Workgroup `index` of a pass over pieces (kTiles = false) or over whole tiles
// (the pass that joins their pieces, kTiles = true).
template <bool kTiles>
__device__ Kv4Item kv4_item(const Kv4AttendArgs& a, int index) {
    const int lane = threadIdx.x & 63, kv = a.cache.kv_heads, seqs = a.batch.seqs;
    const auto load = [&](int s, Kv4Seq& q, int& tiles, int& blocks) {
        tiles = blocks = 0;
        q = Kv4Seq{0, 0, 0};
        if (s >= seqs) return;
        bool bad;
        q = kv4_seq(a.batch, a.cache.page_shift, s, bad);
        if (bad && index == 0 && a.status) raise_status(a.status, kBadBatch);
        tiles = (int)(((int64_t)q.n * a.group + a.tile_rows - 1) / a.tile_rows);
        if (q.n) {
            int b0, b1;
            kv4_blocks(q, a.window, 0, q.n - 1, b0, b1);
            blocks = b1 - b0;
        }
    };
    Kv4Seq q;
    int tiles, blocks;
    int64_t work = 0;
    for (int s0 = 0; s0 < seqs; s0 += kWave) {
        load(s0 + lane, q, tiles, blocks);
        work += (int64_t)tiles * blocks;
    }
    const int64_t share = (wave_sum_i64(work) * kv + (1 << a.slots_log2) - 1) >> a.slots_log2;
    const int piece = __builtin_amdgcn_readfirstlane((int)max((int64_t)a.min_blocks, share));
    Kv4Item it;
    it.live = false;
    it.head = index % kv;
    const int want = index / kv;
    int before = 0, pieces_before = 0;
    for (int s0 = 0; s0 < seqs; s0 += kWave) {
        if (s0 || seqs > kWave) load(s0 + lane, q, tiles, blocks);
        const int splits = blocks <= kKv4Whole ? 1 : (blocks + piece - 1) / piece;
        const int mine = kTiles ? tiles : tiles * splits;
        int upto = mine, pieces = tiles * splits;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int u = __shfl_up(upto, o, kWave), p = __shfl_up(pieces, o, kWave);
            if (lane >= o) upto += u, pieces += p;
        }
        const unsigned long long past = __ballot(before + upto > want);
        if (past) {
            const int who = __ffsll(past) - 1;
            it.seq = s0 + who;
            it.splits = of_lane(splits, who);
            it.row0 = of_lane(q.row0, who);
            it.n = of_lane(q.n, who);
            it.len = of_lane(q.len, who);
            const int at = want - (before + of_lane(upto - mine, who));
            const int first = pieces_before + of_lane(pieces - tiles * splits, who);
            it.tile = kTiles ? at : at / it.splits;
            it.split = kTiles ? 0 : at % it.splits;
            it.first = (first + it.tile * it.splits) * kv + it.head;
            it.live = true;
            return it;
        }
        before += of_lane(upto, kWave - 1);
        pieces_before += of_lane(pieces, kWave - 1);
    }
    return it;
}

}  // namespace dmoe
