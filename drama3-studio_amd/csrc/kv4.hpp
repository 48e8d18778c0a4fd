// The 4-bit paged key/value cache: layout, batch and plan shared by the
// append, read and attention kernels and the C ABI.
//
// A page holds page_size tokens (a power of two, 16..256) of every key/value
// head; a head's part of a page is head_bytes long:
//   key codes    [page_size][D/2] bytes        channel 2j in the low half of byte j
//   value codes  [page_size/4][D/8][4] words   word (a, w, i): token 4a + i, channels 8w..8w+7 from the low bits up
//   key scales   [D/32][page_size] 16-bit words
//   value scales [D/32][page_size] 16-bit words
// A scale word belongs to 32 channels of one token: fp16 bits of the scale s,
// which has at most seven significant bits, so that its four lowest mantissa
// bits are zero, with the zero point z (0..15) in their place.  A code c
// stands for (c - z) s: four bits times seven, exact in fp16, so nothing is
// rounded when a kernel decodes.  Keys lie as rows, because a matrix operand
// takes eight channels of one token; values lie as eight channels of four
// tokens side by side, because there it takes eight tokens of one channel,
// which byte permutes form from two tokens' words.  Scales of neighbouring tokens lie side by side:
// one 8- or 16-byte load brings a lane all it needs.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv4_places.hpp"

namespace dmoe {

constexpr int kKv4Group = 32;          // channels a scale word
constexpr int kKv4Whole = 16;          // blocks up to which a sequence with tiles of many rows, or a batch whose
                                       // table has no more for its tiles of 17..64 rows, is not cut
constexpr int kKv4MaxSeqs = 4096;
constexpr float kKv4Limit = 32640.0f;  // values beyond are stored as this: 15 s = 2 * 32640 is the largest span in fp16

__host__ __device__ inline int64_t kv4_head_bytes(int page_size, int dim) {
    return (int64_t)page_size * (dim + dim / 8);
}

struct Kv4Cache {
    uint8_t* pages;
    int64_t page_stride;  // bytes
    int num_pages, page_shift, kv_heads, dim;
};

struct Kv4Batch {
    const int32_t* table;   // [seqs, table_cols] page of each page_size tokens
    int64_t table_stride;
    const int32_t* lengths; // [seqs] tokens of each sequence, the call's rows among them
    const int32_t* starts;  // [seqs + 1] first row of each sequence; null: row b is sequence b
    int seqs, table_cols, rows, max_rows;
};

struct Kv4Rotary {
    const float* inv_freq;  // [dim / 2]; null: no rotation
    const uint8_t* axis;    // [dim / 2] axis of each frequency; null: axis 0
    const void* positions;  // [axes, rows]; null: the place in the cache
    int64_t axis_stride;
    int positions_dtype, axes, dim, interleaved;
};

struct Kv4Rows {            // [rows, heads, D] bf16 or fp16
    void* p;
    int64_t row_stride, head_stride;  // elements
};

struct Kv4AppendArgs {
    Kv4Cache cache;
    Kv4Batch batch;
    Kv4Rotary rotary;
    Kv4Rows q, q_out, k, v;
    int q_heads, dtype;
    int* status;
};

struct Kv4ReadArgs {
    Kv4Cache cache;
    Kv4Batch batch;
    Kv4Rows k, v;
    int dtype;
    int* status;
};

struct Kv4AttendArgs {
    Kv4Cache cache;
    Kv4Batch batch;
    Kv4Rows q, out;
    int q_heads, group;     // query heads, and how many of them share a key/value head
    int dtype;
    float scale_log2;       // softmax scale * log2(e)
    int window;             // tokens a row sees, 0: all before it
    int slots_log2;         // work is cut for 2^slots_log2 workgroups,
    int min_blocks;         // in pieces of at least this many blocks
    bool cut;               // if at all: without, there is no room for partial sums
    int64_t groups, slots;  // workgroups; places for partial sums
    int tile_rows;          // packed rows (token, head of the group) of a tile
    float* part;            // [slots][tile_rows][D] unnormalised sums of the pieces of a cut tile
    float* part_ml;         // [slots][tile_rows][2] running maximum and sum
    struct Kv4Record* records;  // [seqs * kv_heads] pieces of each tile, where a sequence is one (null: nothing is cut)
    int* status;
};

void launch_kv4_append(const Kv4AppendArgs& a, hipStream_t st);
void launch_kv4_read(const Kv4ReadArgs& a, hipStream_t st);

// Geometry of an attention call: rows of a tile, workgroups, scratch.
struct Kv4Shape {
    bool one_tile;  // a tile holds all rows of a sequence
    bool cut;       // tiles may be cut, and are joined by a second launch
    int tile_rows, slots_log2, min_blocks;
    int64_t tiles;  // most tiles the batch can hold, for one key/value head
    int64_t groups; // workgroups
    int64_t slots;  // partial sums
    size_t part_bytes, ml_bytes, record_bytes;  // multiples of 16
    size_t bytes() const { return part_bytes + ml_bytes + record_bytes; }
};
Kv4Shape kv4_attend_shape(const Kv4Batch& b, int page_size, int kv_heads, int dim, int group);
// Packed rows of a tile of launch_kv4_attend_tiles, and workgroups the work is cut for.
int kv4_tile_rows(int64_t most_rows, int dim);
int kv4_tile_slots_log2(int64_t most_rows, int dim);
void launch_kv4_attend_tiles(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st);
void launch_kv4_attend(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st);

#ifdef __HIPCC__

// A sequence of the batch.  One whose rows do not lie in the caller's buffers
// or whose tokens do not fit its block table is `bad`: it has no rows then, so
// nothing is read or written for it.
struct Kv4Seq {
    int row0, n, len;  // first row, rows, tokens
};

__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Batch& b, int page_shift, int s, bool& bad) {
    Kv4Seq q;
    q.row0 = b.starts ? b.starts[s] : s;
    const int end = b.starts ? b.starts[s + 1] : s + 1;
    q.len = b.lengths[s];
    bad = q.row0 < 0 || end < q.row0 || end > b.rows || end - q.row0 > b.max_rows || q.len < 0 ||
          q.len > ((int64_t)b.table_cols << page_shift);
    q.n = bad ? 0 : end - q.row0;
    if (bad) q.len = 0;
    return q;
}

#endif  // __HIPCC__

}  // namespace dmoe
