// Attention of many rows a sequence (prompts, chunks, proposals) over the
// 4-bit cache.
//
// A workgroup takes a tile of 32 packed rows a row group and walks the blocks
// of 64 tokens that the tile sees.  Its threads decode each block into LDS
// once, as fp16; the waves then share it.  Products are 32x32x16 fp16 MFMAs,
// transposed as in the kernel of few rows: a lane holds everything of one row
// (column = lane % 32) and P goes from the first product's result into the
// second's operand with no exchange; values lie in LDS by channel with their
// tokens in the order which that needs.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "kv4_attend.hpp"

namespace dmoe {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

// RG groups of 32 rows.  TH = 2: two waves each, which take the two halves of
// every block and are joined at the end.  CH = 2: two waves each, which form
// the same scores and add up half the channels (both sums of a head of 256
// channels would not fit a wave's registers).
template <int D_, int RG, int TH, int CH>
struct Tile {
    static constexpr int D = D_, kGroups = RG, kHalves = TH, kSplit = CH;
    static constexpr int kWaves = RG * TH * CH;
    static constexpr int kThreads = kWaves * kWave;
    static constexpr int kRows = RG * 32;
    static constexpr int kTiles = 2 / TH;          // 32-token results of a wave
    static constexpr int kOut = D / 32 / CH;       // 32-channel results
    // 16-byte code pieces of a block: 32 channels of a key token, or 8 channels of 4 value tokens
    static constexpr int kPieces = kKv4Block * D / 32;
    static constexpr int kKeyBytes = kKv4Block * (D * 2 + 16), kValueBytes = D * 144, kStage = kKeyBytes + kValueBytes;
};
template <int D>
using Few = Tile<D, 2, 2, D == 256 ? 2 : 1>;
template <int D>
using Many = Tile<D, D == 256 ? 4 : 8, 1, D == 256 ? 2 : 1>;

// LDS places, in bytes, of 16-byte chunks, so that neither the pieces' stores
// nor the operands' loads meet in a bank: keys [token][D/8] and values
// [channel][8] with a chunk left free behind each row, values' chunks
// exchanged by their row's sixteen.
template <int D>
__host__ __device__ constexpr int key_at(int token, int chunk) {
    return token * (D * 2 + 16) + chunk * 16;
}
__host__ __device__ constexpr int value_at(int channel, int chunk) {
    return channel * 144 + ((chunk ^ channel >> 4) & 7) * 16;
}
// What to add to the place of chunk hi of token r for chunk 2 j + hi of token
// 32 u + r, and to that of channel r for chunk 2 y + hi of channel 32 c + r.
template <int D>
__host__ __device__ constexpr int key_step(int u, int j) {
    return u * 32 * (D * 2 + 16) + j * 32;
}
__host__ __device__ constexpr int value_step(int c, int y) { return c * 32 * 144 + ((y ^ c) & 3) * 32; }

// A byte for each of a block's four 16-token parts, set where the part lies on
// no page; left in LDS by the threads that decode the keys.
typedef uint32_t Parts;
__device__ __forceinline__ uint32_t bad_parts(Parts parts) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)parts); }

// A thread's 16 bytes of key codes and their scale word, or of value codes and
// the scale words of their four tokens; their page, and that of the block after.
struct Piece {
    v4u codes;
    v2u scales;
    int page, next;
};

template <int D>
__device__ __forceinline__ int piece_token(bool is_v, int at) { return is_v ? at / (D / 8) * 4 : at / (D / 32); }

// Where in a page a thread's pieces lie, but for their token.
struct Place {
    int codes, scales;
};
template <int D>
__device__ __forceinline__ Place piece_place(bool is_v, int at, int page_shift) {
    const int size = 1 << page_shift, part = at % (D / 32), word = at % (D / 8);
    return is_v ? Place{size * (D / 2) + word * 16, size * (D + D / 16) + word / 4 * size * 2}
                : Place{part * 16, size * D + part * size * 2};
}

template <int D>
__device__ __forceinline__ void load_page(const Kv4AttendArgs& a, const int32_t* table, bool is_v, int at, int block, int end,
                                          Piece& piece) {
    int token = kv4_token(block, piece_token<D>(is_v, at), end);  // behind the end: the last token's
    // has the page copied before this load: a copy left to the loop's end would wait for the load
    asm("" : "+v"(piece.page), "+v"(token));
    piece.next = *(const int32_t*)((const char*)table + (uint32_t)(token >> a.cache.page_shift) * 4u);
}

template <int D>
__device__ __forceinline__ void load_piece(const Kv4AttendArgs& a, const uint8_t* head, const Place& place, bool is_v, int at,
                                           int block, Piece& piece) {
    // the slot of a value piece's first token: their four lie together, 2 D bytes like keys'
    const uint32_t slot = (block * kKv4Block + piece_token<D>(is_v, at)) & ((1 << a.cache.page_shift) - 1);
    piece.page = piece.next;
    asm("" : "+v"(piece.page));
    const uint32_t page = (unsigned)piece.page >= (unsigned)a.cache.num_pages ? 0u : (unsigned)piece.page;
    const uint8_t* base = head + (int64_t)((uint64_t)page * (uint64_t)a.cache.page_stride);
    piece.codes = *(const v4u*)(base + (slot * (D / 2) + (uint32_t)place.codes));
    const uint8_t* scales = base + (slot * 2 + (uint32_t)place.scales);
    if (is_v) piece.scales = *(const v2u*)scales;
    else piece.scales[0] = *(const uint16_t*)scales;
}

// Notes which of a block's parts lie on no page.
template <int D>
__device__ __forceinline__ void store_page(const Kv4AttendArgs& a, int at, const Piece& piece, Parts& parts) {
    const int token = piece_token<D>(false, at);
    if (at % (D / 32) == 0 && token % 16 == 0) ((uint8_t*)&parts)[token / 16] = (unsigned)piece.page >= (unsigned)a.cache.num_pages;
}

// Decodes a piece into LDS in sixteen steps of a pair of values, so that they
// can stand between products.  Keys and values take the same steps, from
// words x and y that are chosen; a key token's eight channels come to lie in
// the order 0 4 2 6 1 5 3 7, and the query's are laid alike.
template <int D>
struct Decoder {
    Scales s0, s1;
    uint32_t x, y, held;
    int place;

    // keys, values: the places of their stages
    __device__ __forceinline__ Decoder(const Kv4AttendArgs& a, const CodeBits& bits, bool is_v, int at, int block, int lowest,
                                       int end, const Piece& piece, int keys, int values)
        : x(0), y(0), held(0) {
        const int token = piece_token<D>(is_v, at);
        uint32_t w0 = piece.scales[0], w1 = piece.scales[1];
        if (is_v) {
            // slots that hold no token, or one that no row sees, may hold anything; their values must be numbers
            const int kept = (unsigned)piece.page >= (unsigned)a.cache.num_pages ? 0 : kv4_left(block, token, end);
            w0 &= (kept > 0 ? 0xFFFFu : 0u) | (kept > 1 ? 0xFFFF0000u : 0u);
            w1 &= (kept > 2 ? 0xFFFFu : 0u) | (kept > 3 ? 0xFFFF0000u : 0u);
            if (kv4_left(block, 0, lowest) > 0) {
                const int gone = kv4_left(block, token, lowest);
                w0 &= (gone > 0 ? 0u : 0xFFFFu) | (gone > 1 ? 0u : 0xFFFF0000u);
                w1 &= (gone > 2 ? 0u : 0xFFFFu) | (gone > 3 ? 0u : 0xFFFF0000u);
            }
            const int word = at % (D / 8), quad = token / 4;
            // 16 tokens of an operand step: lanes 0..31 take tokens 0..3 and 8..11 of them, lanes 32..63 the others
            place = values + value_at(8 * word, quad / 4 * 2 + (quad & 1)) + (quad >> 1 & 1) * 8;
        } else {
            w0 = w1 = (w0 & 0xFFFFu) | w0 << 16;
            place = keys + key_at<D>(token, 4 * (at % (D / 32)));
        }
        s0 = scales_of(bits, w0);
        s1 = scales_of(bits, w1);
    }

    __device__ __forceinline__ void step(const CodeBits& bits, bool is_v, const Piece& piece, int u, uint8_t* stages) {
        const int b = u / 4, t = u % 4;
        const uint32_t sel = 0x0C000C00u | (4 + b) << 16 | b;
        if (t == 0) x = is_v ? __builtin_amdgcn_perm(piece.codes[1], piece.codes[0], sel) : piece.codes[b];
        if (t == 1) y = is_v ? __builtin_amdgcn_perm(piece.codes[3], piece.codes[2], sel) : piece.codes[b] >> 8;
        const v2h pair = t == 0   ? low_pair(bits, x, s0.low_zero, s0.scale)
                         : t == 1 ? low_pair(bits, y, s1.low_zero, s1.scale)
                         : t == 2 ? high_pair(bits, x, s0.high_zero, s0.scale)
                                  : high_pair(bits, y, s1.high_zero, s1.scale);
        if (t & 1) *(v2u*)(stages + place + (2 * b + t / 2) * (is_v ? 144 : 8)) = v2u{held, __builtin_bit_cast(uint32_t, pair)};
        else held = __builtin_bit_cast(uint32_t, pair);
    }
};

// N products with their operands loaded two ahead (three measure the same and
// take more registers), and beside(i) behind product i: the matrix unit takes
// 32 cycles for one, in which the wave can issue some six vector instructions.
// The compiler left to itself puts the products together and the vector
// instructions behind them.
template <int N, class Load, class Product, class Beside>
__device__ __forceinline__ void products(Load&& load, Product&& product, Beside&& beside) {
    constexpr int kAhead = 2;
    v8h operand[kAhead + 1];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) operand[i] = load(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i + kAhead < N) operand[(i + kAhead) % (kAhead + 1)] = load(i + kAhead);
        product(i, operand[i % (kAhead + 1)]);
        __builtin_amdgcn_sched_barrier(0);
        beside(i);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// What a wave keeps of its 32 rows and does with a block.
template <class T>
struct Rows {
    static constexpr int D = T::D, kSteps = D / 16;
    static constexpr int kScores = T::kTiles * kSteps, kPairs = T::kTiles * 8, kAdds = 2 * T::kTiles * T::kOut;
    const Kv4AttendArgs& a;
    const Kv4Segment& it;
    int lane, r, hi, group, half, split;
    int row_a, row_b;              // the tile's packed rows
    int wave_a, wave_b;            // this wave's, maybe none
    int place;                     // of this lane's token
    int lowest, end;               // the tokens that any row of the tile sees
    int p_first, p_last;           // places of this wave's rows
    v8h query[kSteps];
    float score_scale;             // of the scores in powers of two
    float base, shift;             // the maximum that weights are taken from; 8 - base in powers of two
    float sum;
    bool seen, huge;               // huge: base's product with the scale has lost its digits
    v16f out[T::kOut];
    v8h p[2 * T::kTiles];

    __device__ __forceinline__ Rows(const Kv4AttendArgs& args, const Kv4Segment& seg) : a(args), it(seg) {
        lane = segment_lane();
        r = lane & 31;
        hi = lane >> 5;
        const int wave = wave_index();
        group = wave % T::kGroups;
        half = wave / T::kGroups % T::kHalves;
        split = wave / T::kGroups / T::kHalves;
        const int packed = it.n * a.group;
        row_a = it.row_a;
        row_b = min(row_a + T::kRows, packed);
        wave_a = row_a + 32 * group;
        wave_b = min(wave_a + 32, row_b);
        place = it.len - it.n + min(wave_a + r, packed - 1) / a.group;
        lowest = kv4_lowest(it.len - it.n + row_a / a.group, a.window);
        end = it.len - it.n + (row_b - 1) / a.group + 1;
        p_first = it.len - it.n + wave_a / a.group;
        p_last = it.len - it.n + (wave_b - 1) / a.group;
    }

    // Row `row` of this wave in a tensor of heads.
    __device__ __forceinline__ int64_t row_at(const Kv4Rows& t, int row) const {
        const int packed = min(wave_a + row, it.n * a.group - 1);
        return (int64_t)(it.row0 + packed / a.group) * t.row_stride + (int64_t)(it.head * a.group + packed % a.group) * t.head_stride;
    }

    __device__ __forceinline__ void load_query() {
        const uint16_t* q = (const uint16_t*)a.q.p + row_at(a.q, r) + 8 * hi;
        v4i raw[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) raw[j] = *(const v4i*)(q + 16 * j);
        float most = largest(raw, a.dtype);
        most = fmaxf(most, __shfl_xor(most, 32, kWave));
        score_scale = scale_query(raw, most, a.dtype, a.scale_log2, query);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) query[j] = __builtin_shufflevector(query[j], query[j], 0, 1, 4, 5, 2, 3, 6, 7);
        base = sum = 0.0f;
        shift = kKv4Shift;
        seen = huge = false;
#pragma unroll
        for (int c = 0; c < T::kOut; ++c) out[c] = v16f{};
    }

    __device__ __forceinline__ bool sees(int block) const {
        const int first = block * kKv4Block;
        return wave_a < wave_b && first <= p_last &&
               (a.window <= 0 || (int64_t)first + kKv4Block - 1 > (int64_t)p_first - a.window);
    }

    // Reports entries of the table that name no page, of tokens in the blocks
    // [from, to) which a row of the tile would see.
    __device__ __forceinline__ void report(const int32_t* table, int from, int to) const {
        const int shift = a.cache.page_shift, last = kv4_token(to - 1, kKv4Block - 1, end) >> shift;
        for (int i = (max(from * kKv4Block, lowest) >> shift) + (int)threadIdx.x; i <= last; i += T::kThreads)
            if ((unsigned)table[i] >= (unsigned)a.cache.num_pages) raise_status(a.status, kBadBatch);
    }

    template <class Beside>
    __device__ __forceinline__ void scores(const uint8_t* keys, v16f (&s)[T::kTiles], Beside&& beside) const {
        // results in turn: a product does not wait for the one before it
        const uint8_t* place = keys + key_at<D>(32 * half + r, hi);
        products<kScores>(
            [&](int i) { return *(const v8h*)(place + key_step<D>(i % T::kTiles, i / T::kTiles)); },
            [&](int i, v8h k) {
                v16f& to = s[i % T::kTiles];
                to = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, query[i / T::kTiles], i < T::kTiles ? v16f{} : to, 0, 0, 0);
            },
            beside);
    }

    // Hides the scores of tokens that the rows do not see; `bad`: which of the
    // block's parts lie on no page, a byte each.
    __device__ __forceinline__ void mask(v16f (&s)[T::kTiles], int block, uint32_t bad) const {
        const int first = block * kKv4Block;
        // s[i][x]: token 32 u + 8 (x / 4) + 4 hi + x % 4 of the block
        if (bad || first + kKv4Block - 1 > p_first || (a.window > 0 && first <= (int64_t)p_last - a.window)) {
            const int high = place - first - 4 * hi;
            const int low = a.window > 0 ? (int)max((int64_t)-first, (int64_t)high - a.window + 1) : -first;
#pragma unroll
            for (int i = 0; i < T::kTiles; ++i) {
                const int u = T::kHalves == 1 ? i : half;
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int t = 32 * u + 8 * (x / 4) + x % 4;
                    s[i][x] = ((t > high) | (t < low) | (int)(bad >> (16 * u + x / 8 * 8) & 1)) ? -__builtin_inff() : s[i][x];
                }
            }
        }
    }

    // Adds up the weights that exponentials<false>() has formed from the base
    // there is.  A score so far above it that its weight leaves fp16 shows in their
    // sum; then, and for a row's first tokens, the row's base is brought up to
    // its maximum and they are formed again.  Else no maximum is needed.
    __device__ __forceinline__ void settle(const v16f (&s)[T::kTiles], float part) {
        const bool mine = !seen || huge || !(part < 0x1p22f);
        if (__any(mine)) {
            float top = s[0][0];
#pragma unroll
            for (int i = 0; i < T::kTiles; ++i)
#pragma unroll
                for (int x = 0; x < 16; ++x) top = fmaxf(top, s[i][x]);
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            const bool either = ((int)mine | __shfl_xor((int)mine, 32, kWave)) != 0;  // of the row's two lanes
            if (either && (seen ? top > base : top > -__builtin_inff())) {
                const float fade = seen ? __builtin_amdgcn_exp2f((base - top) * score_scale) : 0.0f;
                base = top;
                shift = kKv4Shift - base * score_scale;
                huge = !(fabsf(shift) <= 0x1p20f);
                seen = true;
                sum *= fade;
#pragma unroll
                for (int c = 0; c < T::kOut; ++c) out[c] *= fade;
            }
            part = __any(huge) ? exponentials<true>(s) : exponentials<false>(s);
        }
        sum += part;
    }

    // P of the scores and this lane's part of its sum, of the weights as they
    // are multiplied.  base * scale is rounded once for all of a row's tokens,
    // the same factor in the weights and in their sum; where that has lost its
    // digits (huge), scores are first taken from the base, which never leaves
    // anything above zero.
    template <bool kHuge>
    __device__ __forceinline__ void pair(const v16f (&s)[T::kTiles], int n, float (&part)[4]) {
        const int i = n / 8, x = n % 8 * 2;
        float t[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            t[y] = __builtin_fmaf(s[i][x + y], score_scale, shift);
            if (kHuge && huge) t[y] = __builtin_fmaf(s[i][x + y] - base, score_scale, kKv4Shift);
        }
        const v2h e{(_Float16)__builtin_amdgcn_exp2f(t[0]), (_Float16)__builtin_amdgcn_exp2f(t[1])};
        part[n % 4] = __builtin_amdgcn_fdot2(e, v2h{(_Float16)1.0f, (_Float16)1.0f}, part[n % 4], false);
        p[2 * i + x / 8][x % 8] = e[0];
        p[2 * i + x / 8][x % 8 + 1] = e[1];
    }
    template <bool kHuge>
    __device__ __forceinline__ float exponentials(const v16f (&s)[T::kTiles]) {
        float part[4] = {};
#pragma unroll
        for (int n = 0; n < kPairs; ++n) pair<kHuge>(s, n, part);
        return (part[0] + part[1]) + (part[2] + part[3]);
    }

    template <class Beside>
    __device__ __forceinline__ void add(const uint8_t* values, Beside&& beside) {
        // a half's steps are 2 and 3: the other bit of (y ^ c) turned over
        const uint8_t* place = values + value_at(r, hi) + split * T::kOut * 32 * 144;
        const int turn = T::kHalves == 1 ? 0 : 64 * half;
        products<kAdds>(
            [&](int i) {
                const int step = value_step(i % T::kOut, i / T::kOut);
                return *(const v8h*)(place + (T::kHalves == 1 ? step : step & 64 ? step - turn : step + turn));
            },
            [&](int i, v8h v) {
                v16f& to = out[i % T::kOut];
                to = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[i / T::kOut], to, 0, 0, 0);
            },
            beside);
    }

    // The maximum that the weights were taken from, in powers of two.
    __device__ __forceinline__ float top() const {
        return !seen ? -__builtin_inff() : huge ? base * score_scale : kKv4Shift - shift;
    }

    __device__ __forceinline__ void store_part(float top) const {
        if (wave_a + r >= row_b || it.slot < 0 || it.slot >= a.slots) return;  // no place: offsets that go back
        const int c0 = 32 * T::kOut * split + 4 * hi;
        const int64_t at = it.slot * a.tile_rows + 32 * group + r;
        float* o = a.part + at * D + c0;
#pragma unroll
        for (int c = 0; c < T::kOut; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *(v4f*)(o + 32 * c + 8 * x) = v4f{out[c][4 * x], out[c][4 * x + 1], out[c][4 * x + 2], out[c][4 * x + 3]};
        if (c0 == 0) *(v2f*)(a.part_ml + at * 2) = v2f{top, sum};
    }

    __device__ __forceinline__ v2u result(int c, int x, float inv) const {
        return v2u{narrow2(out[c][4 * x] * inv, out[c][4 * x + 1] * inv, a.dtype),
                   narrow2(out[c][4 * x + 2] * inv, out[c][4 * x + 3] * inv, a.dtype)};
    }

    __device__ __forceinline__ void store(float top) const {
        if (!it.whole) return store_part(top);
        if (wave_a + r >= row_b) return;
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        uint16_t* o = (uint16_t*)a.out.p + row_at(a.out, r) + 32 * T::kOut * split + 4 * hi;
#pragma unroll
        for (int c = 0; c < T::kOut; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x) *(v2u*)(o + 32 * c + 8 * x) = result(c, x, inv);
    }

    // The same by way of LDS, `kStoreBytes` for each wave, so that whole rows
    // are stored, and past the caches: nine prompts of up to 2000 tokens, 32
    // heads, take 175 us so, 7 us more with eight bytes of 32 rows at a time (33
    // more with those past the caches).
    static constexpr int kRowBytes = 64 * T::kOut + 16, kStoreBytes = 32 * kRowBytes;
    __device__ __forceinline__ void store(float top, uint8_t* lds) const {
        if (!it.whole) return store_part(top);
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        uint8_t* mine = lds + r * kRowBytes + 8 * hi;
#pragma unroll
        for (int c = 0; c < T::kOut; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x) *(v2u*)(mine + 64 * c + 16 * x) = result(c, x, inv);
        constexpr int kChunks = 4 * T::kOut;  // of 16 bytes of a row
#pragma unroll
        for (int i = 0; i < kChunks / 2; ++i) {
            const int row = (i * kWave + lane) / kChunks, chunk = lane % kChunks;
            const v4u x = *(const v4u*)(lds + row * kRowBytes + chunk * 16);
            if (wave_a + row < row_b) __builtin_nontemporal_store(x, (v4u*)((uint16_t*)a.out.p + row_at(a.out, row) + 32 * T::kOut * split + 8 * chunk));
        }
    }
};

template <class T>
struct alignas(16) Stages {
    uint8_t stage[2][T::kStage];  // keys, then values
    Parts parts[2];
};

// A segment of a tile of up to 64 rows: block after block, the next one's
// pieces decoded before the products, with the loads of the one after behind
// them.  12 sequences, 40 packed rows a key/value head of 256 channels, 4096 tokens:
// 27 us, 18 MB.  Two thirds are the start and the end (pages, first pieces,
// partial sums); a further 4096 tokens take 12 us, in which the vector unit is
// the bound, since a block is decoded for few rows.
template <class T>
__device__ __forceinline__ void attend_few(const Kv4AttendArgs& a, const Kv4Segment& it, Stages<T>& lds) {
    constexpr int D = T::D, kMine = 2 * T::kPieces / T::kThreads;  // pieces of a thread, keys then values
    static_assert(kMine * T::kThreads == 2 * T::kPieces && T::kPieces % kWave == 0, "whole waves' pieces of one kind");
    const int from = it.from, to = it.to;
    const int32_t* table = a.batch.table + (int64_t)it.seq * a.batch.table_stride;
    const CodeBits bits = code_bits();
    Rows<T> rows(a, it);
    const uint8_t* head = a.cache.pages + (int64_t)it.head * kv4_head_bytes(1 << a.cache.page_shift, D);
    const Place place[2] = {piece_place<D>(false, (int)threadIdx.x % T::kPieces, a.cache.page_shift),
                            piece_place<D>(true, (int)threadIdx.x % T::kPieces, a.cache.page_shift)};
    Piece piece[kMine];
    const auto each = [&](auto&& f) {
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
            const bool is_v = kMine > 1 ? m >= kMine / 2 : (int)threadIdx.x >= T::kPieces;
            f(is_v, kMine > 1 ? m % (kMine > 1 ? kMine / 2 : 1) * T::kThreads + (int)threadIdx.x : (int)threadIdx.x % T::kPieces, piece[m]);
        }
    };
    const auto load = [&](int block) {
        each([&](bool is_v, int at, Piece& x) { load_piece<D>(a, head, place[is_v], is_v, at, min(block, to - 1), x); });
        each([&](bool is_v, int at, Piece& x) { load_page<D>(a, table, is_v, at, min(block + 1, to - 1), rows.end, x); });
    };
    const auto store = [&](int block) {
        uint8_t* stage = lds.stage[(block - from) & 1];
        each([&](bool is_v, int at, Piece& x) {
            if (!is_v) store_page<D>(a, at, x, lds.parts[(block - from) & 1]);
            Decoder<D> decoder(a, bits, is_v, at, block, rows.lowest, rows.end, x, 0, T::kKeyBytes);
#pragma unroll
            for (int u = 0; u < 16; ++u) decoder.step(bits, is_v, x, u, stage);
        });
    };
    const auto nothing = [](int) {};
    if (from < to) {
        each([&](bool is_v, int at, Piece& x) { x.page = 0, load_page<D>(a, table, is_v, at, from, rows.end, x); });
        load(from);
    }
    rows.load_query();
    if (from < to) {
        store(from);
        load(from + 1);
    }
    for (int block = from; block < to; ++block) {
        lds_barrier();
        const uint8_t* stage = lds.stage[(block - from) & 1];
        const uint32_t bad = bad_parts(lds.parts[(block - from) & 1]);
        if (bad) rows.report(table, block, block + 1);
        if (block + 1 < to) store(block + 1);
        load(block + 2);
        if (rows.sees(block)) {
            v16f s[T::kTiles];
            rows.scores(stage, s, nothing);
            rows.mask(s, block, bad);
            rows.settle(s, rows.template exponentials<false>(s));
            rows.add(stage + T::kKeyBytes, nothing);
        }
    }

    rows.sum += __shfl_xor(rows.sum, 32, kWave);
    float top = rows.top();
    if constexpr (T::kHalves == 2) {
        // the second halves' sums by way of LDS, a lane's values a row of its own length apart
        constexpr int kValues = 16 * T::kOut, kStride = T::kGroups * T::kSplit * kWave;
        static_assert(kStride * (kValues + 2) * 4 <= 2 * T::kStage, "the halves are joined in the stages");
        float* share = (float*)lds.stage + kWave * (rows.group + T::kGroups * rows.split) + rows.lane;
        __syncthreads();
        if (rows.half) {
#pragma unroll
            for (int c = 0; c < T::kOut; ++c)
#pragma unroll
                for (int x = 0; x < 16; ++x) share[(16 * c + x) * kStride] = rows.out[c][x];
            share[kValues * kStride] = top;
            share[(kValues + 1) * kStride] = rows.sum;
        }
        __syncthreads();
        if (rows.half) return;
        const float other = share[kValues * kStride], both = fmaxf(top, other);
        const float f = top == both ? 1.0f : __builtin_amdgcn_exp2f(top - both);
        const float h = other == both ? 1.0f : __builtin_amdgcn_exp2f(other - both);
        rows.sum = f * rows.sum + h * share[(kValues + 1) * kStride];
        top = both;
#pragma unroll
        for (int c = 0; c < T::kOut; ++c)
#pragma unroll
            for (int x = 0; x < 16; ++x) rows.out[c][x] = f * rows.out[c][x] + h * share[(16 * c + x) * kStride];
    }
    rows.store(top);
}

template <class T>
__global__ __launch_bounds__(T::kThreads, 2) void kv4_attend_few_kernel(Kv4AttendArgs a) {
    __shared__ Stages<T> lds;
    Kv4Shares shares(a, blockIdx.x);
    Kv4Segment seg;
    for (bool first = true; shares.next(seg); first = false) {
        if (!first) __syncthreads();  // the segment before has been read
        if (seg.n) attend_few<T>(a, seg, lds);
    }
}

// A piece of a tile of many rows.  Between two barriers a wave forms the
// scores of block b + 1 while it turns those of block b into weights, then
// adds block b up while it decodes its piece of a later block: products
// (matrix unit, LDS) and vector instructions of one wave side by side.  Half
// of the waves decode keys, two blocks ahead, the others values, one ahead;
// two stages of each are enough.
//
// Bound by the vector unit: a block of 64 tokens takes a wave 32 products of
// 32 cycles and some 260 vector instructions, 32 of them exponentials, on a
// unit that two waves share, and keeps LDS busy more than half of the time;
// the matrix unit works 44% of it.  2048 rows behind 14336 tokens, 16
// heads over 2 of 128 channels: 281 us, 917 TFLOP/s.  Two waves in turn, one
// with its products and one with its vector instructions, took 324 us: a
// wave alone issues a vector instruction only every fifth cycle.
template <class T>
__global__ __launch_bounds__(T::kThreads, 2) void kv4_attend_many_kernel(Kv4AttendArgs a) {
    constexpr int D = T::D, kSide = T::kThreads / 2, kMine = (T::kPieces + kSide - 1) / kSide;
    static_assert(T::kWaves == 8 && kMine <= 2, "two waves a SIMD; one or two pieces a thread");
    __shared__ __attribute__((aligned(16))) uint8_t stages[2 * T::kStage];  // two of keys, two of values
    __shared__ __attribute__((aligned(16))) Parts parts[4];
    Kv4Segment it;
    if (!kv4_piece(a, it)) return;
    const int from = it.from, to = it.to;
    const int32_t* table = a.batch.table + (int64_t)it.seq * a.batch.table_stride;
    const CodeBits bits = code_bits();
    Rows<T> rows(a, it);
    const bool is_v = wave_index() >= 4;
    const uint8_t* head = a.cache.pages + (int64_t)it.head * kv4_head_bytes(1 << a.cache.page_shift, D);
    const Place place = piece_place<D>(is_v, (int)threadIdx.x % min(kSide, T::kPieces), a.cache.page_shift);
    Piece piece[kMine];
    const auto each = [&](auto&& f) {
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
            f(m * kSide + (int)threadIdx.x % min(kSide, T::kPieces), piece[m]);  // where there are few, two threads take the same
        }
    };
    const auto load = [&](int block) {
        each([&](int at, Piece& x) { load_piece<D>(a, head, place, is_v, at, min(block, to - 1), x); });
        each([&](int at, Piece& x) { load_page<D>(a, table, is_v, at, min(block + 1, to - 1), rows.end, x); });
    };
    const auto note = [&](int block) {
        if (!is_v) each([&](int at, Piece& x) { store_page<D>(a, at, x, parts[(block - from) & 3]); });
    };
    const auto decoder = [&](int m, int block) {
        const int n = (block - from) & 1;
        return Decoder<D>(a, bits, is_v, m * kSide + (int)threadIdx.x % min(kSide, T::kPieces), block, rows.lowest, rows.end, piece[m],
                          n * T::kKeyBytes, 2 * T::kKeyBytes + n * T::kValueBytes);
    };
    const auto store = [&](int block) {
        note(block);
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
            Decoder<D> d = decoder(m, block);
#pragma unroll
            for (int u = 0; u < 16; ++u) d.step(bits, is_v, piece[m], u, stages);
        }
    };
    const auto nothing = [](int) {};
    int held = from;  // the block of the loaded pieces
    // behind the last block stages of old keys are multiplied and old pieces decoded, for nothing
    Parts bad = 0;
    uint32_t any_bad = 0;
    const auto turn = [&](int block, v16f (&s)[T::kTiles], v16f (&ahead)[T::kTiles]) {
        const uint8_t* next = stages + ((block - from + 1) & 1) * T::kKeyBytes;
        any_bad |= bad_parts(bad);
        rows.mask(s, block, bad_parts(bad));
        bad = parts[(block + 1 - from) & 3];  // the next block's, behind the last one an old one's
        if constexpr (T::kSplit == 1) {
            float part[4] = {};
            rows.scores(next, ahead, [&](int i) {
#pragma unroll
                for (int n = rows.kPairs * i / rows.kScores; n < rows.kPairs * (i + 1) / rows.kScores; ++n)
                    rows.template pair<false>(s, n, part);
            });
            rows.settle(s, (part[0] + part[1]) + (part[2] + part[3]));
        } else {
            rows.settle(s, rows.template exponentials<false>(s));
        }
        note(held);
        const uint8_t* now = stages + 2 * T::kKeyBytes + ((block - from) & 1) * T::kValueBytes;
        Decoder<D> d = decoder(0, held), e = decoder(kMine - 1, held);
        rows.add(now, [&](int i) {
#pragma unroll
            for (int u = 16 * i / rows.kAdds; u < 16 * (i + 1) / rows.kAdds; ++u) {
                d.step(bits, is_v, piece[0], u, stages);
                if constexpr (kMine == 2) e.step(bits, is_v, piece[1], u, stages);
            }
        });
        if constexpr (T::kSplit == 2) rows.scores(next, ahead, nothing);  // no registers for two blocks' scores
        load(++held);
        lds_barrier();
    };
    if (from < to) {
        each([&](int at, Piece& x) { x.page = 0, load_page<D>(a, table, is_v, at, from, rows.end, x); });
        load(held);
    }
    rows.load_query();
    if (from < to) {
        store(held);
        load(++held);
        if (!is_v) {
            store(held);
            load(++held);
        }
        lds_barrier();
        v16f s[T::kTiles];
        bad = parts[0];
        rows.scores(stages, s, nothing);
        if constexpr (T::kSplit == 1) {
            for (int block = from; block < to; ++block) {
                v16f ahead[T::kTiles];
                turn(block, s, ahead);
#pragma unroll
                for (int i = 0; i < T::kTiles; ++i) s[i] = ahead[i];
            }
        } else {
            for (int block = from; block < to; ++block) turn(block, s, s);
        }
    }
    if (any_bad) rows.report(table, from, to);  // here, not at each block: 176 us for nine prompts of up to 2000 tokens, there 180
    rows.sum += __shfl_xor(rows.sum, 32, kWave);
    static_assert(T::kWaves * Rows<T>::kStoreBytes <= sizeof(stages), "results leave through the stages");
    rows.store(rows.top(), stages + wave_index() * Rows<T>::kStoreBytes);  // every wave is behind the last barrier
}

template <int D>
void launch_dim(const Kv4AttendArgs& a, const Kv4Shape& s, hipStream_t st) {
    if (s.one_tile) kv4_attend_few_kernel<Few<D>><<<(unsigned)s.groups, Few<D>::kThreads, 0, st>>>(a);
    else kv4_attend_many_kernel<Many<D>><<<(unsigned)s.groups, Many<D>::kThreads, 0, st>>>(a);
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
