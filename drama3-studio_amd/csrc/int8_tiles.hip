// Products of many rows of 8-bit integers with a matrix of them, in tiles.
//
//   acc[t][n] = sum_k xq[t][k] w[n][k] (int32, exact), out = T(acc xs[t] ws[n] + bias[n] + residual[t][n]),
//   gated: out = T(act(gate) up) of the products with rows n and n + N of w
//
// A workgroup owns TM x TN sums (gated: TN / 2 gate and TN / 2 up rows of the
// matrix, 32 of each in turn, so that a gate's sum and its up's meet in one
// wave); a wave keeps its share in registers and multiplies 32x32x32.  Both
// operands go through LDS, in rings of steps of 128 columns that direct copies
// fill: no register waits for them, and they are asked for a few at a time
// between matrix instructions, one barrier a step.  The sums leave through LDS
// as well, so that a lane finishes eight columns of a row.
//
// 8192 rows, K 4096, N 4096: 109 us a pass, 112 under a tracer, 2.5 POP/s; K
// 12288 with 4096 rows 156 to 169 us, 2.4 to 2.6 (a library's product of 8192
// cubed 2.4).  Power bounds it: with zeros for
// operands the loop takes a quarter less, and matrix instructions alone reach
// 3.5 POP/s on random operands, 5.0 on zeros.  Of a tile's 57 us, 4 are its
// results and 2 its start.  Measured for it: copies asked for all at once behind
// the barrier 5% slower, over a whole step 6%; matrix steps of 64 columns with a
// deeper ring 7%; a third step of rows in the ring, beside two of the matrix, 4%
// faster than two of each; eight waves as fast as four, and 5% faster where few
// tiles run.
#include "int8_epilogue.hpp"
#include "rows8_util.hpp"

namespace dmoe {

namespace {

typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int kTileXcd = 8;         // workgroups go to the XCDs in turn
constexpr int kTileGroup = 4;       // row tiles that are walked together

// One copy of 64 x 16 bytes into LDS: lane l's bytes go to lds + 16 l.  Written
// as an instruction of its own because the compiler waits for every copy
// before the next LDS read; the waits here are tile_wait's.  m0 is written and
// not restored, and named as such; the compiler keeps nothing in it, which is
// what its warning about reserved registers is about.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_to_lds(const uint8_t* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "m0");
}
#pragma clang diagnostic pop

template <int N>
__device__ __forceinline__ void tile_wait() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ __forceinline__ v16i mfma_i8_32(const v4i& a, const v4i& b, const v16i& c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

constexpr int kTileK = 128;         // columns of a step
constexpr int kTileParts = 2;       // of a step's four, over which the copies behind its barrier go out

// TM rows by TN matrix rows a workgroup, WM of its waves along the rows and WN
// along the matrix; rings of SX and SW steps for rows and matrix.
template <int TM_, int TN_, int WM_, int WN_, int SX_, int SW_>
struct Shape {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, SX = SX_, SW = SW_;
    static constexpr int kWaves = WM * WN, kThreads = kWaves * kWave;
};

template <class G, bool GATED>
struct Tile {
    static constexpr int kFM = G::TM / G::WM / 32, kFN = G::TN / G::WN / 32;  // 32-row fragments of a wave
    static_assert(!GATED || kFN % 2 == 0, "a wave has gate and up fragments in turn");
    static constexpr int kChunks = kTileK / 16;
    static constexpr int kUnitX = G::TM * kTileK, kUnitW = G::TN * kTileK;  // bytes of a step
    static constexpr int kRingX = G::SX * kUnitX, kLds = kRingX + G::SW * kUnitW;
    static constexpr int kCopiesX = kUnitX / 1024 / G::kWaves, kCopiesW = kUnitW / 1024 / G::kWaves;  // of a wave for a step
    static constexpr int kCopies = kCopiesX + kCopiesW;
    static constexpr int kCopyRows = 1024 / kTileK;  // rows of a copy
    static constexpr int kSteps = kTileK / 32;       // matrix instructions along a step
    // Behind the barrier of step t, W of step t + SW and then X of step t + SX are asked for.  At that barrier W and X of
    // step t + 1 have to be there; these may still be on their way:
    static_assert(G::SX == G::SW || G::SX == G::SW + 1, "W is the younger of a step's operands");
    static constexpr int kBehind = (G::SW - 2) * kCopies + (G::SX > G::SW ? kCopiesX : 0);
    static constexpr int kCols = GATED ? G::TN / 2 : G::TN;
    static constexpr int kSlots = kTileParts * kFN;  // places of copies between matrix instructions
    // copies [first(p), first(p + 1)) go to place p
    static constexpr int first(int place) { return place * kCopies / kSlots; }
    // waves a SIMD that LDS has room for, in workgroups of at least a wave each
    static constexpr int kPerCu = 160 * 1024 / kLds * G::kWaves / 4, kPerSimd = kPerCu < 1 ? 1 : kPerCu > 2 ? 2 : kPerCu;
    // A chunk's place in its row.  A read of 16 bytes a lane goes by sixteen lanes, whose rows are sixteen different ones
    // modulo 16: two rows fill the banks, and the places of eight pairs differ.
    static_assert(kTileK == 128 && kCopiesX % 2 == 0 && kCopiesW % 2 == 0, "eight chunks a row, copies in pairs");
    static __device__ __forceinline__ int place(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }
};

// With DT kI32 a workgroup takes one of a.splits shares of K and leaves its
// sums to the join.
template <class G, bool GATED, int DT>
__global__ __launch_bounds__(G::kThreads, (Tile<G, GATED>::kPerSimd)) void int8_tile_kernel(Int8Args a, int row_tiles, int col_tiles) {
    using T = Tile<G, GATED>;
    constexpr int FM = T::kFM, FN = T::kFN, BK = kTileK;
    constexpr bool kSplit = DT == kI32;
    __shared__ alignas(1024) uint8_t lds[T::kLds];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    // an XCD takes a contiguous share of the tiles and walks them kTileGroup row tiles at a time, column by column, so
    // that what runs on it at one time shares rows and matrix through its L2
    int m0, n0, split = 0;
    {
        const int total = row_tiles * col_tiles * (kSplit ? a.splits : 1), x = blockIdx.x % kTileXcd, j = blockIdx.x / kTileXcd;
        const int lo = (int)((int64_t)x * total / kTileXcd), hi = (int)((int64_t)(x + 1) * total / kTileXcd);
        if (lo + j >= hi) return;
        int tile = lo + j;
        if constexpr (kSplit) {
            split = tile % a.splits;
            tile /= a.splits;
        }
        const int group = tile / (kTileGroup * col_tiles), at = tile - group * kTileGroup * col_tiles;
        const int wide = min(kTileGroup, row_tiles - group * kTileGroup);
        m0 = (group * kTileGroup + at % wide) * G::TM;
        n0 = at / wide * T::kCols;
    }
    int steps = (a.k + BK - 1) / BK, k0 = 0;
    if constexpr (kSplit) {
        k0 = split * steps / a.splits * BK;
        steps = (split + 1) * steps / a.splits - k0 / BK;
    }
    const int kw = (a.k + 15) / 16 * 16;  // readable columns of a matrix row
    // copies: lane l of copy j brings the chunk that place() wants at its spot, one for even j and one for odd
    uint32_t off_x[T::kCopiesX], off_w[T::kCopiesW];
    const uint32_t src[2] = {T::place(lane / T::kChunks, lane % T::kChunks) * 16u,
                             T::place(lane / T::kChunks + T::kCopyRows, lane % T::kChunks) * 16u};
#pragma unroll
    for (int j = 0; j < T::kCopiesX; ++j) {
        const int row = (wave * T::kCopiesX + j) * T::kCopyRows + lane / T::kChunks;
        off_x[j] = (uint32_t)(min(m0 + row, a.rows - 1) - m0) * (uint32_t)a.xq_stride + src[j % 2];
    }
#pragma unroll
    for (int j = 0; j < T::kCopiesW; ++j) {
        const int row = (wave * T::kCopiesW + j) * T::kCopyRows + lane / T::kChunks;
        int64_t wr;
        if constexpr (GATED) wr = (int64_t)min(n0 + row / 64 * 32 + row % 32, a.n - 1) - n0 + (row & 32 ? a.n : 0);
        else wr = min(n0 + row, a.n - 1) - n0;
        off_w[j] = (uint32_t)(wr * a.w_stride) + src[j % 2];
    }
    // behind a matrix row's last chunk its first of this stage again: the rows hold zeros there
    const int last_k = k0 + (steps - 1) * BK;
    const uint32_t last_back[2] = {last_k + (int)src[0] >= kw ? src[0] : 0u, last_k + (int)src[1] >= kw ? src[1] : 0u};
    const uint8_t* base_x = a.xq + (int64_t)m0 * a.xq_stride + k0;
    const uint8_t* base_w = (const uint8_t*)a.w + (int64_t)n0 * a.w_stride + k0;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const auto copy_x = [&](int step, int slot, int j) {
        copy_to_lds(base_x + (int64_t)step * BK, off_x[j], lds0 + slot * T::kUnitX + (wave * T::kCopiesX + j) * 1024);
    };
    const auto copy_w = [&](int step, int slot, int j) {
        copy_to_lds(base_w + (int64_t)step * BK, off_w[j] - (step == steps - 1 ? last_back[j % 2] : 0u),
                    lds0 + T::kRingX + slot * T::kUnitW + (wave * T::kCopiesW + j) * 1024);
    };
    // operands: lane l holds row l % 32, chunk 2 s + l / 32 of step s
    const int wave_m = wave % G::WM * (FM * 32), wave_n = wave / G::WM;
    const int r = lane % 32, half = lane / 32;
    int at_x[T::kSteps], at_w[T::kSteps];
#pragma unroll
    for (int s = 0; s < T::kSteps; ++s) {
        at_x[s] = (wave_m + r) * BK + T::place(r, 2 * s + half) * 16;
        at_w[s] = (wave_n * FN * 32 + r) * BK + T::place(r, 2 * s + half) * 16 + T::kRingX;
    }
    v4i xf[2][FM], wf[2][FN];
    constexpr int kReading = FN > 1 ? FN / 2 : 1;  // groups of matrix instructions that read the next operands
    const auto read = [&](int to, int slot_x, int slot_w, int s, int g) {
        const uint8_t* px = lds + slot_x * T::kUnitX + at_x[s];
        const uint8_t* pw = lds + slot_w * T::kUnitW + at_w[s];
#pragma unroll
        for (int f = g * FM / kReading; f < (g + 1) * FM / kReading; ++f) xf[to][f] = *(const v4i*)(px + f * 32 * BK);
#pragma unroll
        for (int f = g * FN / kReading; f < (g + 1) * FN / kReading; ++f) wf[to][f] = *(const v4i*)(pw + f * 32 * BK);
    };
    // what the results need is loaded first and held: eight columns of the matrix a lane, the rows' scales
    constexpr int kRaw = FN * 32, kPitch = kRaw + 4;  // sums of a row in LDS, and four ints against bank conflicts
    constexpr int kOut = GATED ? kRaw / 2 : kRaw, kVectors = kOut / 8, kRowsAt = kWave / kVectors;
    static_assert(G::kWaves * (32 * kPitch + FM * 32) * 4 <= T::kLds, "sums and scales fit the ring");
    const int cc = lane % kVectors * 8, n = n0 + wave_n * kOut + cc;
    // column cc of the outputs in a row of sums: gate and up fragments lie in turn
    const int from = GATED ? cc / 32 * 64 + cc % 32 : cc;
    float ws[GATED ? 2 : 1][8], bias[8], xs[(FM + 1) / 2];
    if constexpr (!kSplit) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int ne = min(n + e, a.n - 1);
            ws[0][e] = a.ws[ne];
            if constexpr (GATED) ws[1][e] = a.ws[ne + a.n];
            bias[e] = a.bias ? a.bias[ne] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < (FM + 1) / 2; ++i) xs[i] = a.xs[min(m0 + wave_m + i * kWave + lane, a.rows - 1)];
    }
    v16i acc[FN][FM];  // [matrix fragment][row fragment]: lane l holds row l % 32 and matrix rows 8 (i / 4) + 4 (l / 32) + i % 4
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    // The copies of a step's end, [W of step w, X of step x], from number `from` to `to`.
    const auto copies = [&](int w, int slot_w, int x, int slot_x, int from, int to, auto checked) {
        constexpr bool kChecked = decltype(checked)::value;
#pragma unroll
        for (int c = 0; c < T::kCopies; ++c) {
            if (c < from || c >= to) continue;
            if (c < T::kCopiesW) {
                if (!kChecked || w < steps) copy_w(w, slot_w, c);
            } else {
                if (!kChecked || x < steps) copy_x(x, slot_x, c - T::kCopiesW);
            }
        }
    };
    // The rings' first contents in that order; of the last the first part only, step 0 goes on with it.
    constexpr int kFirst = T::first(FN);
    if constexpr (G::SX > G::SW) copies(0, 0, 0, 0, T::kCopiesW, T::kCopies, std::true_type{});
#pragma unroll
    for (int s = 0; s < G::SW; ++s)
        copies(s, s, s + G::SX - G::SW, s + G::SX - G::SW, 0, s + 1 < G::SW ? T::kCopies : kFirst, std::true_type{});
    if (steps >= G::SX) tile_wait<T::kBehind + kFirst>();
    else tile_wait<0>();
#pragma unroll
    for (int g = 0; g < kReading; ++g) read(0, 0, 0, 0, g);
    // One step of BK columns, and the next one's first operands.  The copies that its barrier frees places for start in
    // its last part and go on in the next step's first ones: a few between matrix instructions, which do not wait for them.
    int slot_x = 0, slot_w = 0;
    const auto step_of = [&](int t, auto tail) {
        constexpr bool kTail = decltype(tail)::value;  // a copy's step may not exist
        const int next_x = slot_x + 1 == G::SX ? 0 : slot_x + 1, before_x = slot_x == 0 ? G::SX - 1 : slot_x - 1;
        const int next_w = slot_w + 1 == G::SW ? 0 : slot_w + 1, before_w = slot_w == 0 ? G::SW - 1 : slot_w - 1;
#pragma unroll
        for (int s = 0; s < T::kSteps; ++s) {
            const bool last = s + 1 == T::kSteps;
            if (last) tile_wait<kTail ? 0 : T::kBehind>();  // every wave has read this step, and the next has come
            const int part = last ? 0 : s + 1;              // of the copies: part 0 is this step's end, the others the last one's
#pragma unroll
            for (int g = 0; g < FN; ++g) {
                if (g < kReading) read((s + 1) % 2, last ? next_x : slot_x, last ? next_w : slot_w, last ? 0 : s + 1, g);
                if (part < kTileParts) {
                    const int from = T::first(part * FN + g), to = T::first(part * FN + g + 1);
                    if (part == 0) copies(t + G::SW, slot_w, t + G::SX, slot_x, from, to, tail);
                    else copies(t - 1 + G::SW, before_w, t - 1 + G::SX, before_x, from, to, tail);
                }
#pragma unroll
                for (int j = 0; j < FM; ++j) acc[g][j] = mfma_i8_32(wf[s % 2][g], xf[s % 2][j], acc[g][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        slot_x = next_x;
        slot_w = next_w;
    };
    int t = 0;
    for (; t + G::SX < steps; ++t) step_of(t, std::false_type{});
    for (; t < steps; ++t) step_of(t, std::true_type{});
    // Every wave is behind its last read of the ring: each takes a part of it and turns its sums over there, 32 rows at
    // a time, so that a lane gets eight columns of a row and the scales, bias and store of whole pieces.
    int* mine = (int*)lds + wave * 32 * kPitch;
    float* mine_xs = (float*)lds + G::kWaves * 32 * kPitch + wave * FM * 32;
    if constexpr (!kSplit) {
#pragma unroll
        for (int i = 0; i < (FM + 1) / 2; ++i)
            if (i * kWave + lane < FM * 32) mine_xs[i * kWave + lane] = xs[i];
    }
    constexpr int kPasses = 32 / kRowsAt;
    const auto put = [&](int j) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(v4i*)(mine + r * kPitch + i * 32 + q * 8 + half * 4) =
                    v4i{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
    };
    const auto sums = [&](int rr, int h, int* raw) {
        *(v4i*)raw = *(const v4i*)(mine + rr * kPitch + from + h * 32);
        *(v4i*)(raw + 4) = *(const v4i*)(mine + rr * kPitch + from + h * 32 + 4);
    };
    if constexpr (kSplit) {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            put(j);
#pragma unroll
            for (int p = 0; p < kPasses; ++p) {
                const int rr = p * kRowsAt + lane / kVectors;
                const int64_t row = m0 + wave_m + j * 32 + rr;
                if (row >= a.rows || n >= a.n) continue;
                int* to = a.part + ((int64_t)split * a.rows + row) * int8_part_cols(a.n, GATED) + n;
#pragma unroll
                for (int h = 0; h < (GATED ? 2 : 1); ++h) {
                    int raw[8];
                    sums(rr, h, raw);
                    *(v4i*)(to + h * int8_part_cols(a.n, false)) = *(v4i*)raw;
                    *(v4i*)(to + h * int8_part_cols(a.n, false) + 4) = *(v4i*)(raw + 4);
                }
            }
        }
    } else {
        const auto values = [&](int j, int rr, float* v, auto checked) {
            constexpr bool kChecked = decltype(checked)::value;
            int raw[GATED ? 2 : 1][8];
#pragma unroll
            for (int h = 0; h < (GATED ? 2 : 1); ++h) sums(rr, h, raw[h]);
            const float by = mine_xs[j * 32 + rr];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = int8_value<kChecked>(raw[0][e], ws[0][e], by);
                if constexpr (GATED) v[e] = int8_gate(v[e], a.gelu) * int8_value<kChecked>(raw[GATED][e], ws[GATED][e], by);
            }
        };
        // The check is asked for a wave at a time: made for every value, it costs 2% of a large product (8192 rows, K 4096,
        // N 4096: 114.0 us, 111.6) and 10% of a ragged one (509 rows, K 2048, N 5003: 18.6 us, 16.9).
        float top = 0.0f;
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(ws[h][e]));
        const bool large = __any(top >= kInt8Large);
        // whole pieces of eight columns: nothing waits for anything but the residual, which is asked for a strip ahead
        const auto whole = [&](auto more) {
            constexpr bool kMore = decltype(more)::value;  // bias or residual
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                float add[kMore ? kPasses : 1][8];
                if (kMore && a.residual) {
#pragma unroll
                    for (int p = 0; p < (kMore ? kPasses : 0); ++p) {
                        const int64_t row = min(m0 + wave_m + j * 32 + p * kRowsAt + lane / kVectors, a.rows - 1);
                        load_cols8<DT>((const char*)a.residual + row * a.residual_stride * elem_bytes<DT>(), n, n + 8, add[p]);
                    }
                }
                put(j);
#pragma unroll
                for (int p = 0; p < kPasses; ++p) {
                    const int rr = p * kRowsAt + lane / kVectors;
                    const int64_t row = m0 + wave_m + j * 32 + rr;
                    float v[8];
                    values(j, rr, v, std::false_type{});
                    if (kMore && a.bias) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] += bias[e];
                    }
                    if (kMore && a.residual) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] += add[kMore ? p : 0][e];
                    }
                    if (row < a.rows) put_cols8<DT>((char*)a.out + (row * a.out_stride + n) * elem_bytes<DT>(), v);
                }
            }
        };
        if (n0 + T::kCols <= a.n && !large) {
            if (a.bias || a.residual) whole(std::true_type{});
            else whole(std::false_type{});
            return;
        }
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            put(j);
#pragma unroll 1
            for (int p = 0; p < kPasses; ++p) {
                const int rr = p * kRowsAt + lane / kVectors;
                const int64_t row = m0 + wave_m + j * 32 + rr;
                if (row >= a.rows || n >= a.n) continue;
                float v[8];
                if (large) values(j, rr, v, std::true_type{});
                else values(j, rr, v, std::false_type{});
                if (a.bias) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += bias[e];
                }
                if (a.residual) {
                    float add[8];
                    load_cols8<DT>((const char*)a.residual + row * a.residual_stride * elem_bytes<DT>(), n, a.n, add);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += add[e];
                }
                store_cols8<DT>((char*)a.out + row * a.out_stride * elem_bytes<DT>(), n, a.n, v);
            }
        }
    }
}

// The shares' sums of eight columns a thread, added up and finished.
template <bool GATED, int DT>
__global__ __launch_bounds__(256) void int8_join_kernel(Int8Args a, int per_row) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (int64_t)a.rows * per_row) return;
    const int64_t row = at / per_row;
    const int n = (int)(at - row * per_row) * 8, cols = int8_part_cols(a.n, GATED);
    const int* p = a.part + row * cols + n;
    // all loads first, also of shares that are not
    v4i part[GATED ? 2 : 1][kInt8MaxSplits][2];
#pragma unroll
    for (int s = 0; s < kInt8MaxSplits; ++s)
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h) {
            const int* q = p + (int64_t)min(s, a.splits - 1) * a.rows * cols + h * (cols / 2);
            part[h][s][0] = *(const v4i*)q;
            part[h][s][1] = *(const v4i*)(q + 4);
        }
    const float by = a.xs[row];
    float v[8], ws[GATED ? 2 : 1][8], bias[8], add[8], top = 0.0f;
#pragma unroll
    for (int h = 0; h < (GATED ? 2 : 1); ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ws[h][e] = a.ws[min(n + e, a.n - 1) + h * a.n];
            top = fmaxf(top, fabsf(ws[h][e]));
        }
    if (a.bias) {
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[e] = a.bias[min(n + e, a.n - 1)];
    }
    if (a.residual) load_cols8<DT>((const char*)a.residual + row * a.residual_stride * elem_bytes<DT>(), n, a.n, add);
    int sum[GATED ? 2 : 1][8] = {};
#pragma unroll
    for (int s = 0; s < kInt8MaxSplits; ++s)
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[h][e] += s < a.splits ? part[h][s][e / 4][e % 4] : 0;
    const auto values = [&](auto checked) {
        constexpr bool kChecked = decltype(checked)::value;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = int8_value<kChecked>(sum[0][e], ws[0][e], by);
            if constexpr (GATED) v[e] = int8_gate(v[e], a.gelu) * int8_value<kChecked>(sum[GATED][e], ws[GATED][e], by);
        }
    };
    if (__any(top >= kInt8Large)) values(std::true_type{});
    else values(std::false_type{});
    if (a.bias) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bias[e];
    }
    if (a.residual) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += add[e];
    }
    store_cols8<DT>((char*)a.out + row * a.out_stride * elem_bytes<DT>(), n, a.n, v);
}

template <class G, bool GATED>
void launch_tiles_of(const Int8Args& a, hipStream_t stream) {
    constexpr int kCols = Tile<G, GATED>::kCols;
    const int64_t row_tiles = (a.rows + G::TM - 1) / G::TM, col_tiles = (a.n + kCols - 1) / kCols;
    const int64_t total = row_tiles * col_tiles * a.splits;
    const dim3 grid((unsigned)((total + kTileXcd - 1) / kTileXcd * kTileXcd)), block(G::kThreads);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a, (int)row_tiles, (int)col_tiles); };
    if (a.splits == 1) {
        if (a.out_dtype == kBF16) go(int8_tile_kernel<G, GATED, kBF16>);
        else if (a.out_dtype == kF16) go(int8_tile_kernel<G, GATED, kF16>);
        else go(int8_tile_kernel<G, GATED, kF32>);
        return;
    }
    if constexpr (G::TN == 64) {
        go(int8_tile_kernel<G, GATED, kI32>);
        const int per_row = (a.n + 7) / 8;
        const dim3 join((unsigned)(((int64_t)a.rows * per_row + 255) / 256));
        const auto end = [&](auto kernel) { hipLaunchKernelGGL(kernel, join, dim3(256), 0, stream, a, per_row); };
        if (a.out_dtype == kBF16) end(int8_join_kernel<GATED, kBF16>);
        else if (a.out_dtype == kF16) end(int8_join_kernel<GATED, kF16>);
        else end(int8_join_kernel<GATED, kF32>);
    }
}

template <class G>
void launch_tiles_as(const Int8Args& a, hipStream_t stream) {
    if (a.gated) launch_tiles_of<G, true>(a, stream);
    else launch_tiles_of<G, false>(a, stream);
}

}  // namespace

void launch_int8_tiles(const Int8Args& a, const Int8Plan& plan, hipStream_t stream) {
    switch (plan.shape) {
        case kInt8Tiles64: return launch_tiles_as<Shape<64, 64, 2, 1, 4, 4>>(a, stream);
        case kInt8Tiles64x128: return launch_tiles_as<Shape<64, 128, 2, 2, 4, 4>>(a, stream);
        case kInt8Tiles128Deep: return launch_tiles_as<Shape<128, 128, 2, 2, 4, 4>>(a, stream);
        case kInt8Tiles128x256: return launch_tiles_as<Shape<128, 256, 2, 4, 3, 3>>(a, stream);
        case kInt8Tiles128: return launch_tiles_as<Shape<128, 128, 2, 2, 2, 2>>(a, stream);
        default: return launch_tiles_as<Shape<256, 256, 2, 4, 3, 2>>(a, stream);
    }
}

}  // namespace dmoe
