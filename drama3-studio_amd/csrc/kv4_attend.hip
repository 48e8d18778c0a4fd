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
//
// Codes become fp16 without conversions: a nibble put into the mantissa of
// 1024 (low) or 64 (high) is 1024 + c or 64 + c, from which 1024 + z or 64 + z
// is taken exactly; times s it is exact again.  Queries are scaled by a power
// of two per row into fp16 (exact), P is shifted by 2^14, which keeps weights
// down to 2^-28 normal, and is rounded to fp16 with the sums in fp32.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "kv4_plan.hpp"

namespace dmoe {
namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr float kShift = 14.0f;  // P is held times 2^14

__device__ __forceinline__ v2h as_h2(uint32_t w) { return __builtin_bit_cast(v2h, w); }

// fp16 pairs of the low (+0) and high (+1) nibbles of w's two low bytes of
// each half, less the zero points, times the scales.
__device__ __forceinline__ v2h low_pair(uint32_t w, v2h zero, v2h scale) {
    return (as_h2((w & 0x000F000Fu) | 0x64006400u) - zero) * scale;
}
__device__ __forceinline__ v2h high_pair(uint32_t w, v2h zero, v2h scale) {
    return (as_h2((w & 0x00F000F0u) | 0x54005400u) - zero) * scale;
}

// The scale words of two tokens (or one, in both halves) as operands of the above.
struct Scales {
    v2h scale, low_zero, high_zero;
};
__device__ __forceinline__ Scales scales_of(uint32_t words) {
    const uint32_t z = words & 0x000F000Fu;
    return Scales{as_h2(words & 0xFFF0FFF0u), as_h2(z | 0x64006400u), as_h2(z << 4 | 0x54005400u)};
}

__device__ __forceinline__ v8h join(v2h a, v2h b, v2h c, v2h d) {
    return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Largest / sum over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float groups_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

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

template <int D>
__device__ __forceinline__ void load_block(const Kv4AttendArgs& a, const int32_t* table, int head, int block, int end,
                                           Raw<D>& raw) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int shift = a.cache.page_shift, size = 1 << shift;
    const int64_t head_at = (int64_t)head * kv4_head_bytes(size, D);
    // tokens behind the last visible one are read from wherever page 0 has them, and masked
    const int kt = block * kKv4Block + 4 * r, vt = block * kKv4Block + 16 * g;
    int kp = kt < end ? table[kt >> shift] : 0, vp = vt < end ? table[vt >> shift] : 0;
    raw.bad = (unsigned)vp >= (unsigned)a.cache.num_pages;
    if ((unsigned)kp >= (unsigned)a.cache.num_pages) kp = 0;
    if (raw.bad) vp = 0;
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

// Pieces of tiles of MT * 16 packed rows (a packed row is a token and one of
// the group's heads); the four waves take every fourth block and are joined
// at the end.
template <int D, int MT>
__global__ __launch_bounds__(kThreads) void kv4_attend_rows_kernel(Kv4AttendArgs a) {
    constexpr int kSteps = D / 32;  // key steps of 32 channels
    constexpr int kOut = D / 16;    // 16-channel results
    constexpr int kParts = Raw<D>::kParts;
    constexpr int kPad = D + 4;
    __shared__ float joined[kWaves][16][kPad];
    __shared__ float join_m[kWaves][MT * 16], join_l[kWaves][MT * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const Kv4Item it = kv4_item<false>(a, blockIdx.x);
    if (!it.live) return;
    const int packed = it.n * a.group, row_a = it.tile * MT * 16, row_b = min(row_a + MT * 16, packed);
    const int i0 = row_a / a.group, i1 = (row_b - 1) / a.group;
    int b0, b1;
    kv4_blocks(Kv4Seq{it.row0, it.n, it.len}, a.window, i0, i1, b0, b1);
    const int64_t blocks = b1 - b0;
    const int from = b0 + (int)(blocks * it.split / it.splits), to = b0 + (int)(blocks * (it.split + 1) / it.splits);
    const int p_first = it.len - it.n + i0, p_last = it.len - it.n + i1, end = p_last + 1;
    const int32_t* table = a.batch.table + (int64_t)it.seq * a.batch.table_stride;

    // this lane's rows: place in the sequence, query operands, scale of the scores
    int place[MT];
    float score_scale[MT];
    v8h query[MT][kSteps];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int pr = min(row_a + 16 * t + r, packed - 1), token = pr / a.group, h = it.head * a.group + pr % a.group;
        place[t] = it.len - it.n + token;
        const uint16_t* q = (const uint16_t*)a.q.p + (int64_t)(it.row0 + token) * a.q.row_stride +
                            (int64_t)h * a.q.head_stride + g * (D / 4);
        v4i raw[kSteps];
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            raw[j] = *(const v4i*)(q + 8 * j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = (uint32_t)raw[j][i];
                const float x = a.dtype == kBF16 ? bf16_to_f32(w & 0xFFFF) : f16_to_f32(w & 0xFFFF);
                const float y = a.dtype == kBF16 ? bf16_to_f32(w >> 16) : f16_to_f32(w >> 16);
                most = fmaxf(most, fmaxf(fabsf(x), fabsf(y)));
            }
        }
        most = groups_max(most);
        int e = 0;
        if (most > 0.0f && most < __builtin_inff()) (void)frexpf(most, &e);
        const float down = ldexpf(1.0f, -max(-120, min(120, e)));
        score_scale[t] = fmaxf(a.scale_log2 * ldexpf(1.0f, max(-120, min(120, e))), 1e-35f);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = (uint32_t)raw[j][i];
                x[2 * i] = (a.dtype == kBF16 ? bf16_to_f32(w & 0xFFFF) : f16_to_f32(w & 0xFFFF)) * down;
                x[2 * i + 1] = (a.dtype == kBF16 ? bf16_to_f32(w >> 16) : f16_to_f32(w >> 16)) * down;
            }
            // the order in which low_pair / high_pair take a word's channels
            query[t][j] = v8h{(_Float16)x[0], (_Float16)x[4], (_Float16)x[1], (_Float16)x[5],
                              (_Float16)x[2], (_Float16)x[6], (_Float16)x[3], (_Float16)x[7]};
        }
    }

    // Scores are held less `base`, the row's running maximum, which the first
    // product starts from: 2^((S - base) scale) never overflows, however large
    // the scores are.
    float base[MT], l[MT];
    bool seen[MT];
    v4f out[MT][kOut];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        base[t] = l[t] = 0.0f;
        seen[t] = false;
#pragma unroll
        for (int j = 0; j < kOut; ++j) out[t][j] = v4f{0, 0, 0, 0};
    }

    for (int block = from + wave; block < to; block += kWaves) {
        Raw<D> raw;
        load_block<D>(a, table, it.head, block, end, raw);
        const bool any_bad = __any(raw.bad);
        if (any_bad && a.status) raise_status(a.status, kBadBatch);

        v4f s[MT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int t = 0; t < MT; ++t) s[t][i] = v4f{-base[t], -base[t], -base[t], -base[t]};
            Scales sc[kParts];
#pragma unroll
            for (int c = 0; c < kParts; ++c) {
                const uint32_t w = raw.key_scale[c][i / 2];
                sc[c] = scales_of(i & 1 ? __builtin_amdgcn_perm(w, w, 0x03020302) : __builtin_amdgcn_perm(w, w, 0x01000100));
            }
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const Scales& c = sc[kParts == 2 ? j / 4 : 0];
                const uint32_t w = key_word<D>(raw, i, j);
                const v8h k = join(low_pair(w, c.low_zero, c.scale), high_pair(w, c.high_zero, c.scale),
                                   low_pair(w >> 8, c.low_zero, c.scale), high_pair(w >> 8, c.high_zero, c.scale));
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, query[t][j], s[t][i], 0, 0, 0);
            }
        }

        // s[t][i][x]: token 16 g + 4 x + i of the block
        const int first = block * kKv4Block;
        const bool whole = !any_bad && first + kKv4Block - 1 <= p_first && (a.window <= 0 || first > p_last - a.window);
        if (!whole) {
            // slots that hold no token may hold anything: a weight of zero
            // times a value that is no number would reach the sum
            const int kept = raw.bad ? 0 : end - first - 16 * g;
#pragma unroll
            for (int c = 0; c < kParts; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int at = 8 * h + 2 * x;
                        raw.value_scale[c][h][x] &= (at < kept ? 0xFFFFu : 0u) | (at + 1 < kept ? 0xFFFF0000u : 0u);
                    }
        }
        v8h p[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (!whole) {
                const int low = a.window > 0 ? (int)max((int64_t)-1, (int64_t)place[t] - a.window) : -1;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int token = first + 16 * g + 4 * x + i;
                        if (raw.bad || token > place[t] || token <= low) s[t][i][x] = -__builtin_inff();
                    }
            }
            float top = s[t][0][0];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) top = fmaxf(top, s[t][i][x]);
            top = groups_max(top);
            const bool up = top > 0.0f || (!seen[t] && top > -__builtin_inff());
            if (__any(up)) {
                const float by = up ? top : 0.0f;
                const float fade = seen[t] ? __builtin_amdgcn_exp2f(-by * score_scale[t]) : 0.0f;
                base[t] += by;
                seen[t] |= up;
                l[t] *= fade;
#pragma unroll
                for (int j = 0; j < kOut; ++j) out[t][j] *= fade;
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] -= by;
            }
            float e[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    e[i][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i][x], score_scale[t], kShift));
                    l[t] += e[i][x];
                }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[t][h][4 * x + i] = (_Float16)e[i][2 * h + x];
        }

#pragma unroll
        for (int c = 0; c < kParts; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Scales sc[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[x] = scales_of(raw.value_scale[c][h][x]);
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
                    const v8h even = join(low_pair(pair[0], sc[0].low_zero, sc[0].scale), low_pair(pair[1], sc[1].low_zero, sc[1].scale),
                                          low_pair(pair[2], sc[2].low_zero, sc[2].scale), low_pair(pair[3], sc[3].low_zero, sc[3].scale));
                    const v8h odd = join(high_pair(pair[0], sc[0].high_zero, sc[0].scale), high_pair(pair[1], sc[1].high_zero, sc[1].scale),
                                         high_pair(pair[2], sc[2].high_zero, sc[2].scale), high_pair(pair[3], sc[3].high_zero, sc[3].scale));
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        out[t][8 * c + 2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, p[t][h], out[t][8 * c + 2 * b], 0, 0, 0);
                        out[t][8 * c + 2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, p[t][h], out[t][8 * c + 2 * b + 1], 0, 0, 0);
                    }
                }
            }
    }

    // the four waves' sums into one
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        l[t] = groups_sum(l[t]);
        if (g == 0) {
            join_m[wave][16 * t + r] = seen[t] ? base[t] * score_scale[t] : -__builtin_inff();
            join_l[wave][16 * t + r] = l[t];
        }
    }
    constexpr int kLanes = D / 8;                // threads of a row, eight channels each
    const int row_in = threadIdx.x / kLanes, c0 = threadIdx.x % kLanes * 8;
    constexpr int kRowsAtOnce = kThreads / kLanes;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (t) __syncthreads();
#pragma unroll
        for (int c = 0; c < kParts; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int j = 0; j < (D == 64 ? 4 : 8); ++j)
                    joined[wave][r][128 * c + (D == 64 ? 4 : 8) * (4 * g + x) + j] = out[t][8 * c + j][x];
        __syncthreads();
        for (int q = row_in; q < 16; q += kRowsAtOnce) {
            const int pr = row_a + 16 * t + q;
            if (pr >= row_b) continue;
            float top = -__builtin_inff(), sum = 0.0f, v[8] = {};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = fmaxf(top, join_m[w][16 * t + q]);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float mw = join_m[w][16 * t + q];
                const float f = mw == top ? 1.0f : __builtin_amdgcn_exp2f(mw - top);
                sum += f * join_l[w][16 * t + q];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(f, joined[w][q][c0 + i], v[i]);
            }
            if (it.splits > 1) {
                const int64_t at = (int64_t)blockIdx.x * a.tile_rows + 16 * t + q;
                *(v4f*)(a.part + at * D + c0) = v4f{v[0], v[1], v[2], v[3]};
                *(v4f*)(a.part + at * D + c0 + 4) = v4f{v[4], v[5], v[6], v[7]};
                if (c0 == 0) *(v2f*)(a.part_ml + at * 2) = v2f{top, sum};
            } else {
                const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
                const int token = pr / a.group, h = it.head * a.group + pr % a.group;
                uint16_t* o = (uint16_t*)a.out.p + (int64_t)(it.row0 + token) * a.out.row_stride + (int64_t)h * a.out.head_stride + c0;
                v4i word;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    word[i] = a.dtype == kBF16 ? (int)(f32_to_bf16(v[2 * i] * inv) | (uint32_t)f32_to_bf16(v[2 * i + 1] * inv) << 16)
                                               : (int)(f32_to_f16(v[2 * i] * inv) | (uint32_t)f32_to_f16(v[2 * i + 1] * inv) << 16);
                *(v4i*)o = word;
            }
        }
    }
}

// Joins the pieces of cut tiles: one row of a tile a workgroup (blockIdx.y),
// the pieces dealt out to the workgroup's rows of threads and added in order.
template <int D>
__global__ __launch_bounds__(kThreads) void kv4_join_kernel(Kv4AttendArgs a) {
    constexpr int kLanes = D / 4;                // threads of a row, four channels each
    constexpr int kAtOnce = kThreads / kLanes;
    __shared__ float sums[kAtOnce][D];
    __shared__ float sum_l[kAtOnce];
    const Kv4Item it = kv4_item<true>(a, blockIdx.x);
    if (!it.live || it.splits == 1) return;
    const int packed = it.n * a.group, pr = it.tile * a.tile_rows + blockIdx.y;
    if (pr >= packed) return;
    const int kv = a.cache.kv_heads, lane_row = threadIdx.x / kLanes, c0 = threadIdx.x % kLanes * 4;
    const auto at = [&](int piece) { return ((int64_t)it.first + (int64_t)piece * kv) * a.tile_rows + blockIdx.y; };
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
    *(v4f*)&sums[lane_row][c0] = v;
    if (c0 == 0) sum_l[lane_row] = sum;
    __syncthreads();
    if (threadIdx.x >= kLanes) return;
    for (int i = 1; i < kAtOnce; ++i) {
        sum += sum_l[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += sums[i][c0 + j];
    }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    const int token = pr / a.group, h = it.head * a.group + pr % a.group;
    uint16_t* o = (uint16_t*)a.out.p + (int64_t)(it.row0 + token) * a.out.row_stride + (int64_t)h * a.out.head_stride + c0;
    uint32_t word[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        word[i] = a.dtype == kBF16 ? f32_to_bf16(v[2 * i] * inv) | (uint32_t)f32_to_bf16(v[2 * i + 1] * inv) << 16
                                   : f32_to_f16(v[2 * i] * inv) | (uint32_t)f32_to_f16(v[2 * i + 1] * inv) << 16;
    *(v2u*)o = v2u{word[0], word[1]};
}

template <int D>
void launch_dim(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    const dim3 grid((unsigned)s.items);
    kv4_attend_rows_kernel<D, 1><<<grid, kThreads, 0, st>>>(a);
    if (s.items > s.tiles * a.cache.kv_heads) {
        const dim3 join((unsigned)(s.tiles * a.cache.kv_heads), a.tile_rows);
        kv4_join_kernel<D><<<join, kThreads, 0, st>>>(a);
    }
}

}  // namespace

Kv4Shape kv4_attend_shape(const Kv4Batch& b, int kv_heads, int dim, int group) {
    Kv4Shape s;
    s.tile_rows = 16;
    s.slots = 1024;
    s.min_blocks = 4;
    const int64_t by_rows = (int64_t)b.rows * group / s.tile_rows + b.seqs;
    const int64_t by_seqs = (int64_t)b.seqs * (((int64_t)b.max_rows * group + s.tile_rows - 1) / s.tile_rows);
    s.tiles = by_rows < by_seqs ? by_rows : by_seqs;
    s.items = s.tiles * kv_heads + s.slots;
    return s;
}

void launch_kv4_attend(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    if (a.cache.dim == 64) launch_dim<64>(a, s, st);
    else if (a.cache.dim == 128) launch_dim<128>(a, s, st);
    else launch_dim<256>(a, s, st);
}

}  // namespace dmoe
