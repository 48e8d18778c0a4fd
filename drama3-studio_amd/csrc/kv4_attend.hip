// Attention of a batch's rows over the 4-bit paged cache.
//
// One pass over keys and values with the running maximum m and sum l of each
// row's softmax: per block of 64 tokens S = K Q^T, P = 2^(S - m), O += V^T P^T.
// Both products are 16x16x32 fp16 MFMAs, kept transposed so that a lane holds
// everything of ONE row in both results (column = lane % 16): the row's scale, maximum
// and sum are plain registers, and P leaves the first product in the lanes
// where the second takes it, with no exchange between lanes.  For that the
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

// A block's bytes of one lane.
template <int D>
struct Raw {
    static constexpr int kKeyWords = D / 32;             // words of each of 4 tokens
    static constexpr int kParts = D == 256 ? 2 : 1;      // 128-channel parts
    v4u key[kKeyWords];                                  // [4 tokens][D / 32] words, in order
    v2u key_scale[kParts];                               // scales of the 4 tokens
    v4u value[kParts][4];                                // words of tokens 4a..4a+3
    v4u value_scale[kParts][2];                          // scales of the 16 tokens
    bool bad;                                            // the 16 value tokens lie on no page
};

// Pages of this lane's four key tokens and 16 value tokens of a block.  Tokens
// behind the last visible one are read from wherever page 0 has them, and masked.
struct Pages {
    int key, value;
};
__device__ __forceinline__ Pages pages_of(const Kv4AttendArgs& a, const int32_t* table, int block, int end) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, shift = a.cache.page_shift;
    const int kt = block * kKv4Block + 4 * r, vt = block * kKv4Block + 16 * g;
    return Pages{kt < end ? table[kt >> shift] : 0, vt < end ? table[vt >> shift] : 0};
}

template <int D>
__device__ __forceinline__ void load_block(const Kv4AttendArgs& a, const Pages& pages, int head, int block, Raw<D>& raw) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int shift = a.cache.page_shift, size = 1 << shift;
    const int64_t head_at = (int64_t)head * kv4_head_bytes(size, D);
    const int kt = block * kKv4Block + 4 * r, vt = block * kKv4Block + 16 * g;
    raw.bad = (unsigned)pages.value >= (unsigned)a.cache.num_pages;
    const int kp = (unsigned)pages.key < (unsigned)a.cache.num_pages ? pages.key : 0, vp = raw.bad ? 0 : pages.value;
    const uint8_t* kb = a.cache.pages + (int64_t)kp * a.cache.page_stride + head_at;
    const uint8_t* vb = a.cache.pages + (int64_t)vp * a.cache.page_stride + head_at;
    const int ks = kt & (size - 1), vs = vt & (size - 1);
    const uint8_t* kc = kb + ks * (D / 2) + g * (D / 8);
    if constexpr (D == 64) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const v2u x = *(const v2u*)(kc + 2 * i * (D / 2)), y = *(const v2u*)(kc + (2 * i + 1) * (D / 2));
            raw.key[i] = v4u{x[0], x[1], y[0], y[1]};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < D / 128; ++c) raw.key[i * (D / 128) + c] = *(const v4u*)(kc + i * (D / 2) + 16 * c);
    }
    const uint8_t* ksc = kb + size * D;
    const uint8_t* vsc = vb + size * D + size * (D / 16);
#pragma unroll
    for (int c = 0; c < Raw<D>::kParts; ++c) {
        const int kgroup = D == 64 ? g / 2 : D == 128 ? g : 2 * g + c;
        raw.key_scale[c] = *(const v2u*)(ksc + (kgroup * size + ks) * 2);
        const int word = D == 64 ? r / 2 : 16 * c + r;
        const uint8_t* vc = vb + size * (D / 2) + (vs / 4 * (D / 8) + word) * 16;
#pragma unroll
        for (int t = 0; t < 4; ++t) raw.value[c][t] = *(const v4u*)(vc + t * (D / 8) * 16);
        const uint8_t* sc = vsc + (word / 4 * size + vs) * 2;
        raw.value_scale[c][0] = *(const v4u*)sc;
        raw.value_scale[c][1] = *(const v4u*)(sc + 16);
    }
}

template <int D>
__device__ __forceinline__ uint32_t key_word(const Raw<D>& raw, int token, int word) {
    const int i = token * (D / 32) + word;
    return raw.key[i / 4][i % 4];
}

// Pieces of tiles of 16 packed rows (a packed row is a token and one of the
// group's heads); the four waves take every fourth block and are joined at
// the end.
template <int D>
__global__ __launch_bounds__(kThreads, D < 256 ? 2 : 1) void kv4_attend_rows_kernel(Kv4AttendArgs a) {
    constexpr int kSteps = D / 32;  // key steps of 32 channels
    constexpr int kOut = D / 16;    // 16-channel results
    constexpr int kParts = Raw<D>::kParts;
    __shared__ float joined[kWaves][16][D + 4];
    __shared__ float join_m[kWaves][16], join_l[kWaves][16];
    const int lane = threadIdx.x & 63, wave = wave_index(), r = lane & 15, g = lane >> 4;
    const Kv4Item it = kv4_item<false>(a, blockIdx.x);
    if (!it.live) return;
    const int packed = it.n * a.group, row_a = it.tile * 16, row_b = min(row_a + 16, packed);
    const int i0 = row_a / a.group, i1 = (row_b - 1) / a.group;
    int b0, b1, from, to;
    kv4_blocks(Kv4Seq{it.row0, it.n, it.len}, a.window, i0, i1, b0, b1);
    kv4_piece(it, b0, b1, from, to);
    const int p_first = it.len - it.n + i0, p_last = it.len - it.n + i1, end = p_last + 1;
    const int32_t* table = a.batch.table + (int64_t)it.seq * a.batch.table_stride;

    // The next block is on its way while one is multiplied, and the pages of
    // the one after it.
    Raw<D> even, odd;
    Pages pages{};
    const auto fetch = [&](int block, Raw<D>& raw) {
        if (block >= to) return;
        load_block<D>(a, pages, it.head, block, raw);
        if (block + kWaves < to) pages = pages_of(a, table, block + kWaves, end);
    };
    if (from + wave < to) {
        pages = pages_of(a, table, from + wave, end);
        fetch(from + wave, even);
    }

    // this lane's row: place in the sequence, query operands, scale of the scores
    const int pr = min(row_a + r, packed - 1), token_in = pr / a.group, head_in = it.head * a.group + pr % a.group;
    const int place = it.len - it.n + token_in;
    v8h query[kSteps];
    float score_scale;
    {
        const uint16_t* q = (const uint16_t*)a.q.p + (int64_t)(it.row0 + token_in) * a.q.row_stride +
                            (int64_t)head_in * a.q.head_stride + g * (D / 4);
        v4i raw[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) raw[j] = *(const v4i*)(q + 8 * j);
        score_scale = scale_query(raw, groups_max(largest(raw, a.dtype)), a.dtype, a.scale_log2, query);
    }

    // Scores are held less `base`, the row's running maximum, which the first
    // product starts from: 2^((S - base) scale) never overflows, however large
    // the scores are.
    float base = 0.0f, sum = 0.0f;
    bool seen = false;
    v4f out[kOut];
#pragma unroll
    for (int j = 0; j < kOut; ++j) out[j] = v4f{0, 0, 0, 0};

    const CodeBits bits = code_bits();
    const auto multiply = [&](int block, Raw<D>& raw) {
        const bool any_bad = __any(raw.bad);
        if (any_bad && a.status) raise_status(a.status, kBadBatch);
        v4f s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = v4f{-base, -base, -base, -base};
            Scales sc[kParts];
#pragma unroll
            for (int c = 0; c < kParts; ++c) {
                const uint32_t w = raw.key_scale[c][i / 2];
                sc[c] = scales_of(bits, __builtin_amdgcn_perm(w, w, i & 1 ? 0x03020302u : 0x01000100u));
            }
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const Scales& c = sc[kParts == 2 ? j / 4 : 0];
                const uint32_t w = key_word<D>(raw, i, j);
                const v8h k = join(low_pair(bits, w, c.low_zero, c.scale), high_pair(bits, w, c.high_zero, c.scale),
                                   low_pair(bits, w >> 8, c.low_zero, c.scale), high_pair(bits, w >> 8, c.high_zero, c.scale));
                s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, query[j], s[i], 0, 0, 0);
            }
        }

        // s[i][x]: token 16 g + 4 x + i of the block
        const int first = block * kKv4Block;
        if (any_bad || first + kKv4Block - 1 > p_first || (a.window > 0 && first <= p_last - a.window)) {
            // tokens 16 g + 0..15 of the block that the row sees: those in [low, high]
            const int at = first + 16 * g;
            const int high = raw.bad ? -1 : place - at;
            const int low = a.window > 0 ? (int)max((int64_t)0, (int64_t)place - a.window + 1 - at) : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    s[i][x] = (4 * x + i > high) | (4 * x + i < low) ? -__builtin_inff() : s[i][x];
            // slots that hold no token may hold anything: a weight of zero
            // times a value that is no number would reach the sum
            const int kept = raw.bad ? 0 : end - at;
#pragma unroll
            for (int c = 0; c < kParts; ++c)
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    raw.value_scale[c][x / 4][x % 4] &= (2 * x < kept ? 0xFFFFu : 0u) | (2 * x + 1 < kept ? 0xFFFF0000u : 0u);
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) top = fmaxf(top, s[i][x]);
        top = groups_max(top);
        const bool up = top > 0.0f || (!seen && top > -__builtin_inff());
        if (__any(up)) {
            const float by = up ? top : 0.0f;
            const float fade = seen ? __builtin_amdgcn_exp2f(-by * score_scale) : 0.0f;
            base += by;
            seen |= up;
            sum *= fade;
#pragma unroll
            for (int j = 0; j < kOut; ++j) out[j] *= fade;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] -= by;
        }
        v8h p[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][2 * h + x], score_scale, kKv4Shift));
                    sum += e;
                    p[h][4 * x + i] = (_Float16)e;
                }
#pragma unroll
        for (int c = 0; c < kParts; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Scales sc[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[x] = scales_of(bits, raw.value_scale[c][h][x]);
                // words of this lane's channels for tokens 8h..8h+7 of its 16
                uint32_t w[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    w[x] = raw.value[c][2 * h + x / 4][x % 4];
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
    };
    for (int block = from + wave; block < to; block += 2 * kWaves) {
        fetch(block + kWaves, odd);
        multiply(block, even);
        if (block + kWaves >= to) break;
        fetch(block + 2 * kWaves, even);
        multiply(block + kWaves, odd);
    }

    // the four waves' sums into one
    sum = groups_sum(sum);
    if (g == 0) {
        join_m[wave][r] = seen ? base * score_scale : -__builtin_inff();
        join_l[wave][r] = sum;
    }
    constexpr int kEach = D == 64 ? 4 : 8;  // neighbouring channels of a lane
#pragma unroll
    for (int c = 0; c < kParts; ++c)
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int j = 0; j < kEach; ++j) joined[wave][r][128 * c + kEach * (4 * g + x) + j] = out[8 * c + j][x];
    __syncthreads();
    constexpr int kLanes = D / 8;  // threads of a row, eight channels each
    const int c0 = threadIdx.x % kLanes * 8;
    for (int q = threadIdx.x / kLanes; q < row_b - row_a; q += kThreads / kLanes) {
        float top = -__builtin_inff(), l = 0.0f, v[8] = {};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, join_m[w][q]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float mw = join_m[w][q];
            const float f = mw == top ? 1.0f : __builtin_amdgcn_exp2f(mw - top);
            l = __builtin_fmaf(f, join_l[w][q], l);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(f, joined[w][q][c0 + i], v[i]);
        }
        if (it.splits > 1) {
            const int64_t at = (int64_t)blockIdx.x * a.tile_rows + q;
            *(v4f*)(a.part + at * D + c0) = v4f{v[0], v[1], v[2], v[3]};
            *(v4f*)(a.part + at * D + c0 + 4) = v4f{v[4], v[5], v[6], v[7]};
            if (c0 == 0) *(v2f*)(a.part_ml + at * 2) = v2f{top, l};
        } else {
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            const int token = (row_a + q) / a.group, h = it.head * a.group + (row_a + q) % a.group;
            uint16_t* o = (uint16_t*)a.out.p + (int64_t)(it.row0 + token) * a.out.row_stride +
                          (int64_t)h * a.out.head_stride + c0;
            *(v4u*)o = v4u{narrow2(v[0] * inv, v[1] * inv, a.dtype), narrow2(v[2] * inv, v[3] * inv, a.dtype),
                           narrow2(v[4] * inv, v[5] * inv, a.dtype), narrow2(v[6] * inv, v[7] * inv, a.dtype)};
        }
    }
}

// Joins the pieces of cut tiles: kJoinRows rows of a tile a workgroup
// (blockIdx.y), a row's pieces dealt out to the threads and added in order.
template <int D>
__global__ __launch_bounds__(kThreads) void kv4_join_kernel(Kv4AttendArgs a, int rows) {
    constexpr int kLanes = D / 4;                // threads of a row, four channels each
    constexpr int kAtOnce = kThreads / kLanes;
    __shared__ float sums[kAtOnce][D];
    __shared__ float sum_l[kAtOnce];
    const Kv4Item it = kv4_item<true>(a, blockIdx.x);
    if (!it.live || it.splits == 1) return;
    const int packed = it.n * a.group, first = it.tile * a.tile_rows;
    const int kv = a.cache.kv_heads, lane_row = threadIdx.x / kLanes, c0 = threadIdx.x % kLanes * 4;
    const int row_end = min((int)(blockIdx.y + 1) * rows, packed - first);
    for (int row = blockIdx.y * rows; row < row_end; ++row) {
        const auto at = [&](int piece) { return ((int64_t)it.first + (int64_t)piece * kv) * a.tile_rows + row; };
        float top = -__builtin_inff();
        for (int i = threadIdx.x & 63; i < it.splits; i += kWave) top = fmaxf(top, a.part_ml[at(i) * 2]);
        top = wave_max(top);
        v4f v = {0, 0, 0, 0};
        float sum = 0.0f;
        for (int i = lane_row; i < it.splits; i += kAtOnce) {
            const v2f ml = *(const v2f*)(a.part_ml + at(i) * 2);
            const float f = ml[0] == top ? 1.0f : __builtin_amdgcn_exp2f(ml[0] - top);
            sum = __builtin_fmaf(f, ml[1], sum);
            const v4f x = *(const v4f*)(a.part + at(i) * D + c0);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(f, x[j], v[j]);
        }
        __syncthreads();  // the row before has been read
        *(v4f*)&sums[lane_row][c0] = v;
        if (c0 == 0) sum_l[lane_row] = sum;
        __syncthreads();
        if (threadIdx.x >= kLanes) continue;
        for (int i = 1; i < kAtOnce; ++i) {
            sum += sum_l[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += sums[i][c0 + j];
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        const int pr = first + row, token = pr / a.group, h = it.head * a.group + pr % a.group;
        uint16_t* o = (uint16_t*)a.out.p + (int64_t)(it.row0 + token) * a.out.row_stride + (int64_t)h * a.out.head_stride + c0;
        *(v2u*)o = v2u{narrow2(v[0] * inv, v[1] * inv, a.dtype), narrow2(v[2] * inv, v[3] * inv, a.dtype)};
    }
}

template <int D>
void launch_dim(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    if (a.tile_rows > 16) launch_kv4_attend_tiles(a, s, st);
    else kv4_attend_rows_kernel<D><<<(unsigned)s.items, kThreads, 0, st>>>(a);
    const int64_t tiles = s.tiles * a.cache.kv_heads;
    if (s.items > tiles) {
        const int most = (int)std::min<int64_t>(a.tile_rows, (int64_t)a.batch.max_rows * a.group);
        const int rows = tiles > 256 ? 32 : 1;
        kv4_join_kernel<D><<<dim3((unsigned)tiles, (most + rows - 1) / rows), kThreads, 0, st>>>(a, rows);
    }
}

}  // namespace

Kv4Shape kv4_attend_shape(const Kv4Batch& b, int page_size, int kv_heads, int dim, int group) {
    Kv4Shape s;
    const int64_t most_rows = (int64_t)b.max_rows * group;
    s.tile_rows = most_rows <= 16 ? 16 : kv4_tile_rows(most_rows, dim);
    s.slots_log2 = most_rows <= 16 ? 9 : kv4_tile_slots_log2(most_rows, dim);
    s.min_blocks = 4;
    const int64_t by_rows = (int64_t)b.rows * group / s.tile_rows + b.seqs;
    const int64_t by_seqs = (int64_t)b.seqs * ((most_rows + s.tile_rows - 1) / s.tile_rows);
    s.tiles = std::min(by_rows, by_seqs);
    // no sequence of a table this narrow is long enough to be cut
    const int64_t most = (int64_t)b.table_cols * page_size / kKv4Block;
    s.items = s.tiles * kv_heads + (most > kKv4Whole ? 1 << s.slots_log2 : 0);
    return s;
}

void launch_kv4_attend(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    if (a.cache.dim == 64) launch_dim<64>(a, s, st);
    else if (a.cache.dim == 128) launch_dim<128>(a, s, st);
    else launch_dim<256>(a, s, st);
}

}  // namespace dmoe
