// Attention of a batch's rows over the 4-bit paged cache.
//
// One pass over keys and values with a base m (a maximum of the row so far)
// and the sum l of each row's softmax: per block of 64 tokens S = K Q^T,
// P = 2^(S - m), O += V^T P^T.  Both products are 16x16x32 fp16 MFMAs, kept
// transposed so that a lane holds everything of ONE row in both results
// (column = lane % 16): the row's scale, base and sum are plain registers, and
// P leaves the first product in the lanes where the second takes it, with no
// exchange between lanes.  For that the
// four 16-token tiles of a block take tokens 4r + i (tile i, operand row r):
// the results of lane group g = lane / 16 are then tokens 16g..16g+15, the
// eight-token slices that the second product's operand wants.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"
#include "kv4_attend.hpp"

namespace dmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

// A block's bytes of one lane: operand row r = lane % 16, lane group g = lane / 16.
template <int D>
struct Keys {
    static constexpr int kParts = D == 256 ? 2 : 1;  // 128-channel parts
    v4u codes[D / 32];                               // tokens 4r..4r+3: D / 32 words each, channels D/4 g and on
    v2u scales[kParts];                              // of the four tokens
};
template <int D>
struct Values {
    static constexpr int kParts = Keys<D>::kParts;
    v4u codes[kParts][4];                            // words of tokens 16g + 4x..+3
    v4u scales[kParts][2];                           // of the 16 tokens
    bool bad;                                        // the tokens lie on no page
};

// Pages of this lane's four key tokens and 16 value tokens of a block.  Tokens
// behind the last one are read from its page, and masked.
struct Pages {
    int key, value;
};
__device__ __forceinline__ Pages pages_of(const Kv4AttendArgs& a, int seq, int block, int end, int r, int g) {
    const int32_t* table = a.batch.table + (int64_t)seq * a.batch.table_stride;
    const int kt = kv4_token(block, 4 * r, end), vt = kv4_token(block, 16 * g, end), shift = a.cache.page_shift;
    return Pages{table[kt >> shift], table[vt >> shift]};
}

// The part of a page that one head has; of page 0 where the table's entry is none.
template <int D>
__device__ __forceinline__ const uint8_t* part_of(const Kv4AttendArgs& a, int page, int head) {
    if ((unsigned)page >= (unsigned)a.cache.num_pages) page = 0;
    return a.cache.pages + (int64_t)((uint64_t)(unsigned)page * (uint64_t)a.cache.page_stride) + (int64_t)head * kv4_head_bytes(1 << a.cache.page_shift, D);
}

template <int D>
__device__ __forceinline__ void load_keys(const Kv4AttendArgs& a, const uint8_t* base, int block, int r, int g, Keys<D>& keys) {
    const int size = 1 << a.cache.page_shift;
    const int slot = (block * kKv4Block + 4 * r) & (size - 1);
    const uint8_t* codes = base + slot * (D / 2) + g * (D / 8);
    if constexpr (D == 64) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const v2u x = *(const v2u*)(codes + 2 * i * (D / 2)), y = *(const v2u*)(codes + (2 * i + 1) * (D / 2));
            keys.codes[i] = v4u{x[0], x[1], y[0], y[1]};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < D / 128; ++c) keys.codes[i * (D / 128) + c] = *(const v4u*)(codes + i * (D / 2) + 16 * c);
    }
#pragma unroll
    for (int c = 0; c < Keys<D>::kParts; ++c) {
        const int group = D == 64 ? g / 2 : D == 128 ? g : 2 * g + c;
        keys.scales[c] = *(const v2u*)(base + size * D + (group * size + slot) * 2);
    }
}

template <int D>
__device__ __forceinline__ void load_values(const Kv4AttendArgs& a, const uint8_t* base, int block, int r, int g, Values<D>& values) {
    const int size = 1 << a.cache.page_shift;
    const int slot = (block * kKv4Block + 16 * g) & (size - 1);
#pragma unroll
    for (int c = 0; c < Values<D>::kParts; ++c) {
        const int word = D == 64 ? r / 2 : 16 * c + r;
        const uint8_t* codes = base + size * (D / 2) + (slot / 4 * (D / 8) + word) * 16;
#pragma unroll
        for (int x = 0; x < 4; ++x) values.codes[c][x] = *(const v4u*)(codes + x * (D / 8) * 16);
        const uint8_t* scales = base + size * D + size * (D / 16) + (word / 4 * size + slot) * 2;
        values.scales[c][0] = *(const v4u*)scales;
        values.scales[c][1] = *(const v4u*)(scales + 16);
    }
}

template <int D>
__device__ __forceinline__ uint32_t key_word(const Keys<D>& keys, int token, int word) {
    const int i = token * (D / 32) + word;
    return keys.codes[i / 4][i % 4];
}

// A share of blocks a wave, a tile of up to 16 packed rows a sequence (a packed
// row is a token and one of the group's heads).  Waves work alone, with no LDS
// and no barrier.  Registers hold one block: its keys are replaced by the next
// one's as soon as the scores are formed, its values when they have been
// added, across segments too, so loads are always on their way.  A head of 256
// channels takes 300 registers for that: one wave a SIMD and half the shares
// (16 sequences of 8000 tokens, 16 heads over 2: 35 us; two waves spill, 55 us).
//
// 32 heads over 8 of 128 channels: 131072 tokens of one sequence take 36 us,
// 151 MB at 4.2 TB/s, as many more 30 us (5.1 TB/s); 64 sequences, 120 MB,
// 38 us.  What is lost is the start (lengths, then pages, then codes, each
// read behind the other) and waits: two waves a SIMD keep the vector unit busy
// two thirds of the time -- 430 of a block's 700 instructions decode its codes
// -- and wait for loads 37% of it.  Three waves spill (60 us for the one sequence),
// twice as many shares add to the start (62 us with the join instead of 51).
template <int D>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void kv4_attend_rows_kernel(Kv4AttendArgs a) {
    constexpr int kSteps = D / 32;  // key steps of 32 channels
    constexpr int kOut = D / 16;    // 16-channel results
    constexpr int kParts = Keys<D>::kParts;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const CodeBits bits = code_bits();

    Kv4Shares shares(a, blockIdx.x * kWaves + wave_index());
    Kv4Segment it, ahead{};
    if (!shares.next(it)) return;
    Keys<D> keys;
    Values<D> values;
    Pages pages{};       // of the block after the loaded one
    bool loaded = false; // the segment's first block of this wave is
    v4i raw_query[kSteps];
    const auto load_query = [&](const Kv4Segment& s) {
        const int pr = min(r, max(s.n * a.group, 1) - 1), token = pr / a.group, head = s.head * a.group + pr % a.group;
        const uint16_t* q = (const uint16_t*)a.q.p + (int64_t)(s.row0 + token) * a.q.row_stride +
                            (int64_t)head * a.q.head_stride + g * (D / 4);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) raw_query[j] = *(const v4i*)(q + 8 * j);
    };
    if (it.n) load_query(it);

    for (;;) {
        const bool more = shares.next(ahead);
        const int packed = it.n * a.group, from = it.from, to = it.to;
        const int p_first = it.len - it.n, p_last = it.len - 1;
        const int place = p_first + min(r, max(packed, 1) - 1) / a.group;
        const bool goes_on = more && ahead.from < ahead.to;
        const auto pages_at = [&](int block) {  // also of the next segment's blocks, as if they lay behind this one's
            const bool here = block < to || !goes_on;
            return pages_of(a, here ? it.seq : ahead.seq, here ? block : ahead.from + block - to, here ? it.len : ahead.len, r, g);
        };
        if (!loaded && from < to) {
            const Pages now = pages_of(a, it.seq, from, it.len, r, g);
            pages = pages_at(from + 1);
            load_keys<D>(a, part_of<D>(a, now.key, it.head), from, r, g, keys);
            load_values<D>(a, part_of<D>(a, now.value, it.head), from, r, g, values);
            values.bad = (unsigned)now.value >= (unsigned)a.cache.num_pages;
        } else if (from + 1 == to) {
            pages = pages_at(to);  // what follows a single block was not known before
        }

        v8h query[kSteps];
        const float score_scale = scale_query(raw_query, groups_max(largest(raw_query, a.dtype)), a.dtype, a.scale_log2, query);
        // Weights are taken from `base`, a maximum of the row so far or less than
        // 2^8 times below one; `shift` is 8 less base in powers of two, `huge` says
        // that base's product with the scale has lost its digits.
        float base = 0.0f, shift = kKv4Shift, sum = 0.0f;
        bool seen = false, huge = false;
        v4f out[kOut];
#pragma unroll
        for (int j = 0; j < kOut; ++j) out[j] = v4f{0, 0, 0, 0};

        for (int block = from; block < to; ++block) {
            const bool any_bad = __any(values.bad);
            if (any_bad && a.status && __any(values.bad && block * kKv4Block + 16 * g + 15 >= kv4_lowest(p_first, a.window)))
                raise_status(a.status, kBadBatch);  // a page that a row would see
            v4f s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = v4f{0, 0, 0, 0};
                Scales sc[kParts];
#pragma unroll
                for (int c = 0; c < kParts; ++c) {
                    const uint32_t w = keys.scales[c][i / 2];
                    sc[c] = scales_of(bits, __builtin_amdgcn_perm(w, w, i & 1 ? 0x03020302u : 0x01000100u));
                }
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    const Scales& c = sc[kParts == 2 ? j / 4 : 0];
                    const uint32_t w = key_word<D>(keys, i, j);
                    const v8h k = join(low_pair(bits, w, c.low_zero, c.scale), high_pair(bits, w, c.high_zero, c.scale),
                                       low_pair(bits, w >> 8, c.low_zero, c.scale), high_pair(bits, w >> 8, c.high_zero, c.scale));
                    s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, query[j], s[i], 0, 0, 0);
                }
            }
            // The next block, in this segment or the one after it.  The last one of
            // all is loaded once more: a load that only some blocks have would be
            // waited for in all of them.
            const bool here = block + 1 < to || !goes_on;
            const int next_head = here ? it.head : ahead.head, next_block = here ? min(block + 1, to - 1) : ahead.from;
            load_keys<D>(a, part_of<D>(a, pages.key, next_head), next_block, r, g, keys);

            // s[i][x]: token 16 g + 4 x + i of the block
            v4u scales[kParts][2];
#pragma unroll
            for (int c = 0; c < kParts; ++c) scales[c][0] = values.scales[c][0], scales[c][1] = values.scales[c][1];
            const int first = block * kKv4Block;
            if (any_bad || first + kKv4Block - 1 > p_first || (a.window > 0 && first <= p_last - a.window)) {
                // tokens 16 g + 0..15 of the block that the row sees: those in [low, high]
                const int at = first + 16 * g;
                const int high = values.bad ? -1 : place - at;
                const int low = a.window > 0 ? (int)max((int64_t)0, (int64_t)place - a.window + 1 - at) : 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        s[i][x] = ((4 * x + i > high) | (4 * x + i < low)) ? -__builtin_inff() : s[i][x];
                // slots that hold no token, or one that no row sees, may hold anything: a
                // weight of zero times a value that is no number would reach the sum
                const int kept = values.bad ? 0 : it.len - at, gone = kv4_lowest(p_first, a.window) - at;
#pragma unroll
                for (int c = 0; c < kParts; ++c)
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        scales[c][x / 4][x % 4] &= (((2 * x < kept) & (2 * x >= gone)) ? 0xFFFFu : 0u) |
                                                   (((2 * x + 1 < kept) & (2 * x + 1 >= gone)) ? 0xFFFF0000u : 0u);
            }
            // P and this lane's part of its sum, of the weights as they are
            // multiplied.  base * scale is rounded once for all of a row's tokens;
            // where that is too rough, scores are first taken from the base.
            v8h p[2];
            const auto weights = [&](bool rough) {
                float part[2] = {};
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            float t[2];
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const float score = s[i + y][2 * h + x];
                                t[y] = __builtin_fmaf(score, score_scale, shift);
                                if (rough && huge) t[y] = __builtin_fmaf(score - base, score_scale, kKv4Shift);
                            }
                            const v2h e{(_Float16)__builtin_amdgcn_exp2f(t[0]), (_Float16)__builtin_amdgcn_exp2f(t[1])};
                            part[x] = __builtin_amdgcn_fdot2(e, v2h{(_Float16)1.0f, (_Float16)1.0f}, part[x], false);
                            p[h][4 * x + i] = e[0];
                            p[h][4 * x + i + 1] = e[1];
                        }
                return part[0] + part[1];
            };
            // A score so far above the base that its weight leaves fp16 shows in
            // the sum; then, and for a row's first tokens, the base is brought up
            // to the maximum.  Else no maximum is needed.
            float part = weights(false);
            const bool mine = !seen || huge || !(part < 0x1p20f);
            if (__any(mine)) {
                float top = s[0][0];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) top = fmaxf(top, s[i][x]);
                top = groups_max(top);
                int either = (int)mine | __shfl_xor((int)mine, 16, kWave);
                either |= __shfl_xor(either, 32, kWave);
                if (either && (seen ? top > base : top > -__builtin_inff())) {
                    const float fade = seen ? __builtin_amdgcn_exp2f((base - top) * score_scale) : 0.0f;
                    base = top;
                    shift = kKv4Shift - base * score_scale;
                    huge = !(fabsf(shift) <= 0x1p20f);
                    seen = true;
                    sum *= fade;
#pragma unroll
                    for (int j = 0; j < kOut; ++j) out[j] *= fade;
                }
                part = __any(huge) ? weights(true) : weights(false);
            }
            sum += part;
#pragma unroll
            for (int c = 0; c < kParts; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    Scales sc[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[x] = scales_of(bits, scales[c][h][x]);
                    // words of this lane's channels for tokens 8h..8h+7 of its 16
                    uint32_t w[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        w[x] = values.codes[c][2 * h + x / 4][x % 4];
                        if constexpr (D == 64) w[x] = r & 1 ? w[x] >> 16 : w[x];
                    }
#pragma unroll
                    for (int b = 0; b < (D == 64 ? 2 : 4); ++b) {
                        uint32_t pair[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            pair[x] = __builtin_amdgcn_perm(w[2 * x + 1], w[2 * x], 0x0C000C00u | (4 + b) << 16 | b);
                        const v8h lower = join(low_pair(bits, pair[0], sc[0].low_zero, sc[0].scale),
                                               low_pair(bits, pair[1], sc[1].low_zero, sc[1].scale),
                                               low_pair(bits, pair[2], sc[2].low_zero, sc[2].scale),
                                               low_pair(bits, pair[3], sc[3].low_zero, sc[3].scale));
                        const v8h upper = join(high_pair(bits, pair[0], sc[0].high_zero, sc[0].scale),
                                               high_pair(bits, pair[1], sc[1].high_zero, sc[1].scale),
                                               high_pair(bits, pair[2], sc[2].high_zero, sc[2].scale),
                                               high_pair(bits, pair[3], sc[3].high_zero, sc[3].scale));
                        const int o = 8 * c + 2 * b;
                        out[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lower, p[h], out[o], 0, 0, 0);
                        out[o + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(upper, p[h], out[o + 1], 0, 0, 0);
                    }
                }
            // The pages after are loaded behind the last use of these: a copy of
            // theirs left to the loop's end would wait for every load.
            int64_t base = part_of<D>(a, pages.value, next_head) - a.cache.pages;
            values.bad = (unsigned)pages.value >= (unsigned)a.cache.num_pages;
            int after = block + 2;
            asm("" : "+v"(base), "+s"(after));
            pages = pages_at(after);
            load_values<D>(a, a.cache.pages + base, next_block, r, g, values);
        }
        loaded = from < to && goes_on;
        if (more && ahead.n) load_query(ahead);

        // lane (r, g) has channels 8 (4 g + x) .. + 7 of row r (D = 64: 4 of them) for x = 0..3
        sum = groups_sum(sum);
        constexpr int kEach = D == 64 ? 4 : 8;
        if (r < packed && !it.whole) {
            const int64_t at = it.slot * a.tile_rows + r;
            float* o = a.part + at * D + 4 * kEach * g;
#pragma unroll
            for (int c = 0; c < kParts; ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int j = 0; j < kEach; j += 4)
                        *(v4f*)(o + 128 * c + kEach * x + j) = v4f{out[8 * c + j][x], out[8 * c + j + 1][x], out[8 * c + j + 2][x], out[8 * c + j + 3][x]};
            if (g == 0) *(v2f*)(a.part_ml + at * 2) = v2f{!seen ? -__builtin_inff() : huge ? base * score_scale : kKv4Shift - shift, sum};
        } else if (r < packed) {
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
            const int token = r / a.group, head = it.head * a.group + r % a.group;
            uint16_t* o = (uint16_t*)a.out.p + (int64_t)(it.row0 + token) * a.out.row_stride +
                          (int64_t)head * a.out.head_stride + 4 * kEach * g;
#pragma unroll
            for (int c = 0; c < kParts; ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int j = 0; j < kEach; j += 4)
                        *(v2u*)(o + 128 * c + kEach * x + j) =
                            v2u{narrow2(out[8 * c + j][x] * inv, out[8 * c + j + 1][x] * inv, a.dtype),
                                narrow2(out[8 * c + j + 2][x] * inv, out[8 * c + j + 3][x] * inv, a.dtype)};
        }
        if (!more) return;
        it = ahead;
    }
}

// Joins the partial sums of cut tiles.  A workgroup has kThreads / (D / 4)
// rows of threads, four channels a thread.  kRowEach: each is another row of
// the tile and adds its pieces in order; else all deal the pieces of one row
// out among them, and LDS brings them together.  Pieces are taken four at a
// time, their loads before their sums, scaled to the largest maximum so far.
template <int D, bool kOneTile, bool kRowEach, int kThreads>
__global__ __launch_bounds__(kThreads) void kv4_join_kernel(Kv4AttendArgs a, int rows) {
    constexpr int kLanes = D / 4, kAtOnce = kThreads / kLanes;
    const int kv = a.cache.kv_heads;
    int pieces, head, row0, n, row_a;
    int64_t first, step, odd;  // slots of the first piece and between them, and what the first lies behind that
    int64_t group = 0;         // of the last piece
    if constexpr (kOneTile) {
        const Kv4Record rec = a.records[blockIdx.x];
        pieces = rec.pieces;
        head = blockIdx.x % kv;
        row0 = rec.row0;
        n = rec.n;
        row_a = 0;
        first = 2 * (int64_t)rec.first;
        step = 2;
        odd = 1;
    } else {
        const Kv4Item it = kv4_item<true>(a, blockIdx.x);
        if (!it.live) return;
        pieces = it.splits;
        head = it.head;
        row0 = it.row0;
        n = it.n;
        row_a = it.tile * a.tile_rows;
        first = it.slot;
        step = kv;
        odd = 0;
        group = it.first + (pieces - 1) * step;
    }
    const int lane_row = threadIdx.x / kLanes, c0 = threadIdx.x % kLanes * 4;
    if (pieces <= 1) return;
    // offsets that go back can name more rows than there are: such tiles' pieces have no place or no workgroup
    if (first < 0 || first + (pieces - 1) * step + odd >= a.slots || group < 0 || group >= a.groups) return;
    const int row_b = min(a.tile_rows, n * a.group - row_a);
    int row = kRowEach ? (int)blockIdx.y * rows + lane_row : (int)blockIdx.y;
    const int row_end = kRowEach ? min(row_b, ((int)blockIdx.y + 1) * rows) : min(row_b, row + 1);
    for (; row < row_end; row += kAtOnce) {
        float top = -__builtin_inff(), sum = 0.0f;
        v4f v = {0, 0, 0, 0};
        constexpr int kBy = kRowEach ? 1 : kAtOnce;
        for (int i = kRowEach ? 0 : lane_row; i < pieces; i += 4 * kBy) {
            v2f ml[4];
            v4f x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int piece = min(i + u * kBy, pieces - 1);
                const int64_t at = (first + piece * step + (piece ? 0 : odd)) * a.tile_rows + row;
                ml[u] = *(const v2f*)(a.part_ml + at * 2);
                x[u] = *(const v4f*)(a.part + at * D + c0);
            }
            float now = top;
#pragma unroll
            for (int u = 0; u < 4; ++u) now = fmaxf(now, ml[u][0]);
            const float fade = top == now ? 1.0f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= fade;
            v *= fade;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (i + u * kBy >= pieces) break;
                const float f = ml[u][0] == now ? 1.0f : __builtin_amdgcn_exp2f(ml[u][0] - now);
                sum = __builtin_fmaf(f, ml[u][1], sum);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(f, x[u][j], v[j]);
            }
        }
        if constexpr (!kRowEach) {
            __shared__ float sums[kAtOnce][D];
            __shared__ float sum_m[kAtOnce], sum_l[kAtOnce];
            *(v4f*)&sums[lane_row][c0] = v;
            if (c0 == 0) {
                sum_m[lane_row] = top;
                sum_l[lane_row] = sum;
            }
            __syncthreads();
            if (lane_row) return;  // of one row only
            float most = top;
#pragma unroll
            for (int i = 1; i < kAtOnce; ++i) most = fmaxf(most, sum_m[i]);
            const float f = top == most ? 1.0f : __builtin_amdgcn_exp2f(top - most);
            sum *= f;
            v *= f;
#pragma unroll 8
            for (int i = 1; i < kAtOnce; ++i) {
                const float h = sum_m[i] == most ? 1.0f : __builtin_amdgcn_exp2f(sum_m[i] - most);
                sum = __builtin_fmaf(h, sum_l[i], sum);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(h, sums[i][c0 + j], v[j]);
            }
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        const int pr = row_a + row, token = pr / a.group, h = head * a.group + pr % a.group;
        uint16_t* o = (uint16_t*)a.out.p + (int64_t)(row0 + token) * a.out.row_stride + (int64_t)h * a.out.head_stride + c0;
        *(v2u*)o = v2u{narrow2(v[0] * inv, v[1] * inv, a.dtype), narrow2(v[2] * inv, v[3] * inv, a.dtype)};
    }
}

template <int D>
void launch_dim(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    if (a.tile_rows > 16) launch_kv4_attend_tiles(a, s, st);
    else kv4_attend_rows_kernel<D><<<(unsigned)s.groups, kThreads, 0, st>>>(a);
    if (!s.cut) return;
    const unsigned tiles = (unsigned)((s.one_tile ? (int64_t)a.batch.seqs : s.tiles) * a.cache.kv_heads);
    const unsigned rows = (unsigned)std::min<int64_t>(a.tile_rows, (int64_t)a.batch.max_rows * a.group);
    // rows of a workgroup where each has threads of its own: more where there are many tiles, few of which may be
    // cut (1200 tiles, none cut: 128 rows 2 us less than 64, 256 rows 4 us, but a cut tile's rows follow each other)
    const unsigned each = tiles > 512 ? 128 : kThreads / (D / 4);
    const dim3 row_each(tiles, (rows + each - 1) / each);
    // few rows: many pieces each, and few workgroups unless there are many tiles; a workgroup a row while that does
    // not fill the chip (12 sequences with 40 rows: 29 us with the attention, 32 with four rows a workgroup)
    if (a.tile_rows <= 16 && tiles <= 32) kv4_join_kernel<D, true, false, 1024><<<dim3(tiles, rows), 1024, 0, st>>>(a, 1);
    else if (a.tile_rows <= 16 || (s.one_tile && (int64_t)tiles * rows <= 4096)) kv4_join_kernel<D, true, false, kThreads><<<dim3(tiles, rows), kThreads, 0, st>>>(a, 1);
    else if (s.one_tile) kv4_join_kernel<D, true, true, kThreads><<<row_each, kThreads, 0, st>>>(a, each);
    else kv4_join_kernel<D, false, true, kThreads><<<row_each, kThreads, 0, st>>>(a, each);
}

}  // namespace

Kv4Shape kv4_attend_shape(const Kv4Batch& b, int page_size, int kv_heads, int dim, int group) {
    Kv4Shape s{};
    // Up to 16 packed rows go to waves that work alone, up to 64 to workgroups
    // that decode a block once for all of them, more to tiles of 128 or 256.
    // One sequence of 131072 tokens with 4 packed rows: 51 us so, 88 us with the
    // workgroups of 64; 12 sequences with 20 rows: 41 us, 72 us with the tiles.
    const int64_t most_rows = (int64_t)b.max_rows * group;
    s.tile_rows = most_rows <= 16 ? 16 : kv4_tile_rows(most_rows, dim);
    // shares of few rows: the waves that the chip holds
    s.slots_log2 = most_rows > 16 ? kv4_tile_slots_log2(most_rows, dim) : dim == 256 ? 10 : 11;
    s.one_tile = most_rows <= 64;  // the kernel of many rows cuts into tiles also where one would do
    // a wave of few rows has little more to do for two blocks than for one; a
    // tile of many rows shorter than kKv4Whole is not worth joining
    const int64_t most_blocks = ((int64_t)b.table_cols * page_size + kKv4Block - 1) / kKv4Block;
    const bool waves = most_rows <= 16;
    s.min_blocks = waves ? 2 : 4;
    s.cut = most_blocks > (waves ? s.min_blocks : kKv4Whole);
    if (!s.cut) s.min_blocks = std::max(s.min_blocks, (int)most_blocks);
    const int64_t by_rows = (int64_t)b.rows * group / s.tile_rows + b.seqs;
    const int64_t by_seqs = (int64_t)b.seqs * ((most_rows + s.tile_rows - 1) / s.tile_rows);
    s.tiles = std::min(by_rows, by_seqs);
    const int64_t cuts = (int64_t)1 << s.slots_log2;
    // shares: as many as wanted, or one a sequence and head where nothing is cut
    const int64_t shares = s.cut ? cuts : std::max(cuts, (int64_t)b.seqs * kv_heads);
    s.groups = !s.one_tile ? s.tiles * kv_heads + (s.cut ? cuts : 0) : waves ? (shares + kWaves - 1) / kWaves : shares;
    // Partial sums: two for each share that there can be.  Of many rows only cut tiles have them, and a tile is cut if
    // its blocks are more than a piece, which has at least a workgroup's average work: less than two pieces a workgroup.
    const int64_t most_shares = (int64_t)b.seqs * kv_heads * ((most_blocks + s.min_blocks - 1) / s.min_blocks);
    s.slots = !s.cut ? 0 : s.one_tile ? 2 * std::min(cuts, most_shares) : std::min(s.groups, 2 * cuts);
    s.part_bytes = (size_t)s.slots * s.tile_rows * dim * sizeof(float);
    s.ml_bytes = (size_t)s.slots * s.tile_rows * 2 * sizeof(float);
    s.record_bytes = s.cut && s.one_tile ? (size_t)b.seqs * kv_heads * sizeof(Kv4Record) : 0;
    // counts of blocks are kept in 31 bits
    if (std::max(most_blocks, (int64_t)s.min_blocks) * s.tiles * kv_heads > INT32_MAX / 2) s.groups = 0;
    return s;
}

void launch_kv4_attend(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    if (a.cache.dim == 64) launch_dim<64>(a, s, st);
    else if (a.cache.dim == 128) launch_dim<128>(a, s, st);
    else launch_dim<256>(a, s, st);
}

}  // namespace dmoe
