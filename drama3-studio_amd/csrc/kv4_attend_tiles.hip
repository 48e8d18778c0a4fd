// Attention of many rows a sequence (prompts, chunks) over the 4-bit cache.
//
// A workgroup takes a tile of 32 packed rows a wave and walks the blocks of 64
// tokens that the tile sees.  All threads decode a block into LDS once, as
// fp16, while the block before it is multiplied; the waves then share it.
// Products are 32x32x16 fp16 MFMAs, transposed as in the kernel of few rows: a
// lane holds everything of one row (column = lane % 32) and P goes from the
// first product's result into the second's operand with no exchange; values
// lie in LDS by channel with their tokens in the order which that needs.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "kv4_attend.hpp"

namespace dmoe {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

// RG groups of 32 rows; with TH = 2 each has two waves, which take the two
// halves of every block and are joined at the end.
template <int D_, int RG, int TH>
struct Tile {
    static constexpr int D = D_, kGroups = RG, kHalves = TH;
    static constexpr int kWaves = RG * TH;
    static constexpr int kThreads = kWaves * kWave;
    static constexpr int kRows = RG * 32;
    // 16-byte code pieces of a block: 32 channels of a key token, or 8 channels of 4 value tokens
    static constexpr int kPieces = kKv4Block * D / 32;
    static constexpr int kMine = (2 * kPieces + kThreads - 1) / kThreads;  // pieces of a thread, keys then values
    static constexpr int kKeyBytes = kKv4Block * D * 2, kStage = 2 * kKeyBytes;
};
template <int D>
using Few = Tile<D, 2, 2>;
template <int D>
using Many = Tile<D, D == 256 ? 4 : 8, 1>;

// LDS places, in bytes, of 16-byte chunks, exchanged so that neither the
// pieces' stores nor the operands' loads meet in a bank: keys [token][D/8],
// values [channel][8].
template <int D>
__device__ __forceinline__ int key_at(int token, int chunk) {
    return token * (D * 2) + ((chunk ^ (D == 64 ? (token >> 1) & 7 : token & 15)) << 4);
}
__device__ __forceinline__ int value_at(int channel, int chunk) {
    return channel * 128 + ((chunk ^ ((channel >> 3) ^ channel)) & 7) * 16;
}

struct Piece {
    v4u codes;
    v2u scales;  // keys: the word in the first half; values: of four tokens
};

// Loads this thread's pieces of a block.
template <class T>
__device__ __forceinline__ void load_pieces(const Kv4AttendArgs& a, const int32_t* table, int head, int block, int end,
                                            Piece (&piece)[T::kMine]) {
    constexpr int D = T::D;
    const int shift = a.cache.page_shift, size = 1 << shift;
    const int64_t head_at = (int64_t)head * kv4_head_bytes(size, D);
#pragma unroll
    for (int m = 0; m < T::kMine; ++m) {
        const int id = threadIdx.x + m * T::kThreads;
        const bool is_v = id >= T::kPieces;
        const int at = is_v ? id - T::kPieces : id;
        if (T::kMine * T::kThreads > 2 * T::kPieces && at >= T::kPieces) continue;
        const int token = block * kKv4Block + (is_v ? at / (D / 8) * 4 : at / (D / 32));
        int page = token < end ? table[token >> shift] : -1;
        const bool none = (unsigned)page >= (unsigned)a.cache.num_pages;
        const uint8_t* base = a.cache.pages + (none ? 0 : (int64_t)page * a.cache.page_stride) + head_at;
        const int slot = token & (size - 1);
        const uint8_t* scales = base + size * D;
        if (is_v) {
            const int word = at % (D / 8);
            piece[m].codes = *(const v4u*)(base + size * (D / 2) + (slot / 4 * (D / 8) + word) * 16);
            piece[m].scales = *(const v2u*)(scales + size * (D / 16) + (word / 4 * size + slot) * 2);
            // slots that hold no token may hold anything; their values must be numbers
            const int kept = none ? 0 : end - token;
            if (kept < 4) {
                piece[m].scales[0] &= (kept > 0 ? 0xFFFFu : 0u) | (kept > 1 ? 0xFFFF0000u : 0u);
                piece[m].scales[1] &= kept > 2 ? 0xFFFFu : 0u;
            }
        } else {
            const int part = at % (D / 32);
            piece[m].codes = *(const v4u*)(base + slot * (D / 2) + part * 16);
            piece[m].scales[0] = none ? 0 : *(const uint16_t*)(scales + (part * size + slot) * 2);
        }
    }
}

// Decodes them into an LDS stage.
template <class T>
__device__ __forceinline__ void store_pieces(const CodeBits& bits, const Piece (&piece)[T::kMine], uint8_t* stage) {
    constexpr int D = T::D;
#pragma unroll
    for (int m = 0; m < T::kMine; ++m) {
        const int id = threadIdx.x + m * T::kThreads;
        const bool is_v = id >= T::kPieces;
        const int at = is_v ? id - T::kPieces : id;
        if (T::kMine * T::kThreads > 2 * T::kPieces && at >= T::kPieces) continue;
        if (is_v) {
            uint8_t* values = stage + T::kKeyBytes;
            const int word = at % (D / 8), quad = at / (D / 8);
            // 16 tokens of an operand step: lanes 0..31 take tokens 0..3 and 8..11 of them, lanes 32..63 the others
            const int chunk = quad / 4 * 2 + (quad & 1), half = (quad >> 1 & 1) * 8;
            const Scales s0 = scales_of(bits, piece[m].scales[0]), s1 = scales_of(bits, piece[m].scales[1]);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t sel = 0x0C000C00u | (4 + b) << 16 | b;
                const uint32_t x = __builtin_amdgcn_perm(piece[m].codes[1], piece[m].codes[0], sel);
                const uint32_t y = __builtin_amdgcn_perm(piece[m].codes[3], piece[m].codes[2], sel);
                const int c = 8 * word + 2 * b;
                *(v2u*)(values + value_at(c, chunk) + half) =
                    v2u{__builtin_bit_cast(uint32_t, low_pair(bits, x, s0.low_zero, s0.scale)),
                        __builtin_bit_cast(uint32_t, low_pair(bits, y, s1.low_zero, s1.scale))};
                *(v2u*)(values + value_at(c + 1, chunk) + half) =
                    v2u{__builtin_bit_cast(uint32_t, high_pair(bits, x, s0.high_zero, s0.scale)),
                        __builtin_bit_cast(uint32_t, high_pair(bits, y, s1.high_zero, s1.scale))};
            }
        } else {
            const int token = at / (D / 32), part = at % (D / 32);
            const uint32_t word = piece[m].scales[0] & 0xFFFFu;
            const Scales s = scales_of(bits, word | word << 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = piece[m].codes[j];
                *(v8h*)(stage + key_at<D>(token, 4 * part + j)) =
                    join(low_pair(bits, w, s.low_zero, s.scale), high_pair(bits, w, s.high_zero, s.scale),
                         low_pair(bits, w >> 8, s.low_zero, s.scale), high_pair(bits, w >> 8, s.high_zero, s.scale));
            }
        }
    }
}

template <class T>
__device__ __forceinline__ void attend_tile(const Kv4AttendArgs& a, const Kv4Segment& it, uint8_t (&lds)[2][T::kStage]) {
    constexpr int D = T::D, kSteps = D / 16, kOut = D / 32, kTiles = 2 / T::kHalves;
    static_assert(T::kHalves == 1 || T::kRows * (D + 2) * 4 <= 2 * T::kStage, "the halves are joined in the stages");
    const int lane = segment_lane(), r = lane & 31, hi = lane >> 5;
    const int wave = wave_index() % T::kGroups, half = wave_index() / T::kGroups;
    const int packed = it.n * a.group, from = it.from, to = it.to;
    const int row_a = it.row_a, row_b = min(row_a + T::kRows, packed);
    const int end = it.len - it.n + (row_b - 1) / a.group + 1;
    const int32_t* table = a.batch.table + (int64_t)it.seq * a.batch.table_stride;
    const CodeBits bits = code_bits();
    Piece piece[T::kMine];
    if (from < to) load_pieces<T>(a, table, it.head, from, end, piece);

    const int wave_a = row_a + 32 * wave, wave_b = min(wave_a + 32, row_b);  // this wave's rows, maybe none
    const int pr = wave_a + r;
    const int token = min(pr, packed - 1) / a.group, head = it.head * a.group + min(pr, packed - 1) % a.group;
    const int place = it.len - it.n + token;
    const int p_first = it.len - it.n + wave_a / a.group, p_last = it.len - it.n + (wave_b - 1) / a.group;
    v8h query[kSteps];
    float score_scale;
    {
        const uint16_t* q = (const uint16_t*)a.q.p + (int64_t)(it.row0 + token) * a.q.row_stride +
                            (int64_t)head * a.q.head_stride + 8 * hi;
        v4i raw[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) raw[j] = *(const v4i*)(q + 16 * j);
        float most = largest(raw, a.dtype);
        most = fmaxf(most, __shfl_xor(most, 32, kWave));
        score_scale = scale_query(raw, most, a.dtype, a.scale_log2, query);
    }

    const float slack = kKv4Slack / score_scale;
    float base = 0.0f, sum = 0.0f;  // as in the kernel of few rows: scores are held less `base`
    bool seen = false;
    v16f out[kOut];
#pragma unroll
    for (int c = 0; c < kOut; ++c) out[c] = v16f{};

    if (from < to) {
        store_pieces<T>(bits, piece, lds[0]);
        load_pieces<T>(a, table, it.head, min(from + 1, to - 1), end, piece);
    }
    for (int block = from; block < to; ++block) {
        __syncthreads();
        const uint8_t* stage = lds[(block - from) & 1];
        const int first = block * kKv4Block;
        // which of the block's four 16-token parts lie on no page
        const int part_token = first + 16 * (lane & 3);
        const bool off = part_token < end && (unsigned)table[part_token >> a.cache.page_shift] >= (unsigned)a.cache.num_pages;
        const uint32_t bad = (uint32_t)__ballot(off) & 15u;
        if (bad && a.status) raise_status(a.status, kBadBatch);
        const bool some = wave_a < wave_b && first <= p_last &&
                          (a.window <= 0 || (int64_t)first + kKv4Block - 1 > (int64_t)p_first - a.window);
        if (some) {
            v16f s[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const int u = T::kHalves == 1 ? i : half;
                const float start = -base;
#pragma unroll
                for (int x = 0; x < 16; ++x) s[i][x] = start;
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    const v8h k = *(const v8h*)(stage + key_at<D>(32 * u + r, 2 * j + hi));
                    s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, query[j], s[i], 0, 0, 0);
                }
            }
            // s[i][x]: token 32 u + 8 (x / 4) + 4 hi + x % 4 of the block
            if (bad || first + kKv4Block - 1 > p_first || (a.window > 0 && first <= (int64_t)p_last - a.window)) {
                const int high = place - first - 4 * hi;
                const int low = a.window > 0 ? (int)max((int64_t)-first, (int64_t)high - a.window + 1) : -first;
#pragma unroll
                for (int i = 0; i < kTiles; ++i) {
                    const int u = T::kHalves == 1 ? i : half;
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int t = 32 * u + 8 * (x / 4) + x % 4;
                        s[i][x] = (t > high) | (t < low) | (bad >> (2 * u + x / 8) & 1) ? -__builtin_inff() : s[i][x];
                    }
                }
            }
            float top = s[0][0];
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int x = 0; x < 16; ++x) top = fmaxf(top, s[i][x]);
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            const bool up = top > slack || (!seen && top > -__builtin_inff());
            if (__any(up)) {
                const float by = up ? top : 0.0f;
                const float fade = seen ? __builtin_amdgcn_exp2f(-by * score_scale) : 0.0f;
                base += by;
                seen |= up;
                sum *= fade;
#pragma unroll
                for (int c = 0; c < kOut; ++c) out[c] *= fade;
#pragma unroll
                for (int i = 0; i < kTiles; ++i) s[i] -= by;
            }
            v8h p[2 * kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][x], score_scale, kKv4Shift));
                    sum += e;
                    p[2 * i + x / 8][x % 8] = (_Float16)e;
                }
#pragma unroll
            for (int c = 0; c < kOut; ++c)
#pragma unroll
                for (int y = 0; y < 2 * kTiles; ++y) {
                    const int step = T::kHalves == 1 ? y : 2 * half + y;
                    const v8h v = *(const v8h*)(stage + T::kKeyBytes + value_at(32 * c + r, 2 * step + hi));
                    out[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[y], out[c], 0, 0, 0);
                }
        }
        if (block + 1 < to) {
            store_pieces<T>(bits, piece, lds[(block + 1 - from) & 1]);
            load_pieces<T>(a, table, it.head, min(block + 2, to - 1), end, piece);
        }
    }

    sum += __shfl_xor(sum, 32, kWave);
    float top = seen ? base * score_scale : -__builtin_inff();
    if constexpr (T::kHalves == 2) {
        // the second halves' sums by way of LDS, a lane's values a row of its own length apart
        constexpr int kStride = T::kGroups * kWave;
        float* share = (float*)lds + 64 * wave + lane;
        __syncthreads();
        if (half) {
#pragma unroll
            for (int c = 0; c < kOut; ++c)
#pragma unroll
                for (int x = 0; x < 16; ++x) share[(16 * c + x) * kStride] = out[c][x];
            share[D / 2 * kStride] = top;
            share[(D / 2 + 1) * kStride] = sum;
        }
        __syncthreads();
        if (half) return;
        const float other = share[D / 2 * kStride], both = fmaxf(top, other);
        const float f = top == both ? 1.0f : __builtin_amdgcn_exp2f(top - both);
        const float h = other == both ? 1.0f : __builtin_amdgcn_exp2f(other - both);
        sum = f * sum + h * share[(D / 2 + 1) * kStride];
        top = both;
#pragma unroll
        for (int c = 0; c < kOut; ++c)
#pragma unroll
            for (int x = 0; x < 16; ++x) out[c][x] = f * out[c][x] + h * share[(16 * c + x) * kStride];
    }
    if (pr >= row_b) return;
    if (!it.whole) {
        const int64_t at = it.slot * a.tile_rows + 32 * wave + r;
        float* o = a.part + at * D + 4 * hi;
#pragma unroll
        for (int c = 0; c < kOut; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *(v4f*)(o + 32 * c + 8 * x) = v4f{out[c][4 * x], out[c][4 * x + 1], out[c][4 * x + 2], out[c][4 * x + 3]};
        if (hi == 0) *(v2f*)(a.part_ml + at * 2) = v2f{top, sum};
        return;
    }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    uint16_t* o = (uint16_t*)a.out.p + (int64_t)(it.row0 + token) * a.out.row_stride + (int64_t)head * a.out.head_stride + 4 * hi;
#pragma unroll
    for (int c = 0; c < kOut; ++c)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *(v2u*)(o + 32 * c + 8 * x) = v2u{narrow2(out[c][4 * x] * inv, out[c][4 * x + 1] * inv, a.dtype),
                                              narrow2(out[c][4 * x + 2] * inv, out[c][4 * x + 3] * inv, a.dtype)};
}

template <class T>
__global__ __launch_bounds__(T::kThreads, T::D == 256 ? 1 : 2) void kv4_attend_tiles_kernel(Kv4AttendArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][T::kStage];
    if constexpr (T::kHalves == 2) {
        Kv4Shares shares(a, blockIdx.x);
        Kv4Segment seg;
        for (bool first = true; shares.next(seg); first = false) {
            if (!first) __syncthreads();  // the segment before has been read
            if (seg.n) attend_tile<T>(a, seg, lds);
        }
    } else {
        Kv4Segment seg;
        if (kv4_piece(a, seg)) attend_tile<T>(a, seg, lds);
    }
}

template <int D>
void launch_dim(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    if (a.tile_rows == Few<D>::kRows) kv4_attend_tiles_kernel<Few<D>><<<(unsigned)s.groups, Few<D>::kThreads, 0, st>>>(a);
    else kv4_attend_tiles_kernel<Many<D>><<<(unsigned)s.groups, Many<D>::kThreads, 0, st>>>(a);
}

}  // namespace

int kv4_tile_rows(int64_t most_rows, int dim) {
    if (most_rows <= Few<64>::kRows) return Few<64>::kRows;
    return dim == 256 ? Many<256>::kRows : Many<128>::kRows;
}
int kv4_tile_slots_log2(int64_t most_rows, int dim) { return most_rows <= Few<64>::kRows && dim < 256 ? 9 : 8; }

void launch_kv4_attend_tiles(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    if (a.cache.dim == 64) launch_dim<64>(a, s, st);
    else if (a.cache.dim == 128) launch_dim<128>(a, s, st);
    else launch_dim<256>(a, s, st);
}

}  // namespace dmoe
