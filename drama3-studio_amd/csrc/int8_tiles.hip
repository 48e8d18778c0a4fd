// Products of many rows of 8-bit integers with a matrix of them, in tiles.
//
//   acc[t][n] = sum_k xq[t][k] w[n][k] (int32, exact), out = T(acc xs[t] ws[n] + bias[n] + residual[t][n]),
//   gated: out = T(act(gate) up) of the products with rows n and n + N of w
//
// A workgroup of four waves owns B x B sums (gated: B / 2 gate and B / 2 up
// rows of the matrix against B rows, 32 of each in turn, so that a gate's sum
// and its up's meet in one lane); a wave owns a quarter in registers and
// multiplies 32x32x32.  Both operands go through LDS in a ring of stages of BK
// columns, filled by direct copies that no register waits for.
#include <algorithm>

#include "int8_epilogue.hpp"
#include "rows8_util.hpp"

namespace dmoe {

namespace {

typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int kTileXcd = 8;         // workgroups go to the XCDs in turn
constexpr int kTileGroup = 4;       // row tiles that are walked together

// One copy of 64 x 16 bytes into LDS: lane l's bytes go to lds + 16 l.  Written
// as an instruction of its own because the compiler waits for every copy
// before the next LDS read; the waits here are tile_wait's.
__device__ __forceinline__ void copy_to_lds(const uint8_t* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base));
}

template <int N>
__device__ __forceinline__ void tile_wait() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ __forceinline__ v16i mfma_i8_32(const v4i& a, const v4i& b, const v16i& c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

template <int B, int BK, int S, bool GATED>
struct Tile {
    static constexpr int kF = B / 64;              // 32-row fragments of a wave and side
    static constexpr int kChunks = BK / 16;
    static constexpr int kUnit = B * BK;           // bytes of one side's stage
    static constexpr int kCopies = kUnit / 4096;   // copies of a wave for it
    static constexpr int kCopyRows = 1024 / BK;    // rows of a copy
    static constexpr int kSteps = BK / 32;         // matrix instructions along a stage
    static constexpr int kCols = GATED ? B / 2 : B;
    // a chunk's place in its row: eight lanes of consecutive rows and one chunk fall on all banks
    static __device__ __forceinline__ int place(int row, int chunk) {
        return BK == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3);
    }
};

template <int B, int BK, int S, bool GATED>
__global__ __launch_bounds__(256, B == 256 ? 1 : 2) void int8_tile_kernel(Int8Args a, int row_tiles, int col_tiles) {
    using T = Tile<B, BK, S, GATED>;
    constexpr int F = T::kF;
    __shared__ alignas(1024) uint8_t lds[S * 2 * T::kUnit];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    // an XCD takes a contiguous share of the tiles and walks them kTileGroup row tiles at a time, column by column, so
    // that what runs on it at one time shares rows and matrix through its L2
    int m0, n0;
    {
        const int total = row_tiles * col_tiles, x = blockIdx.x % kTileXcd, j = blockIdx.x / kTileXcd;
        const int lo = (int)((int64_t)x * total / kTileXcd), hi = (int)((int64_t)(x + 1) * total / kTileXcd);
        if (lo + j >= hi) return;
        const int tile = lo + j, group = tile / (kTileGroup * col_tiles), at = tile - group * kTileGroup * col_tiles;
        const int wide = min(kTileGroup, row_tiles - group * kTileGroup);
        m0 = (group * kTileGroup + at % wide) * B;
        n0 = at / wide * T::kCols;
    }
    const int steps = (a.k + BK - 1) / BK;
    const int kw = (a.k + 15) / 16 * 16;  // readable columns of a matrix row
    // copies: lane l of copy j brings the chunk that place() wants at its spot
    uint32_t off_x[T::kCopies], off_w[T::kCopies];
    const int chunk_of = lane % T::kChunks;
    int src[T::kCopies];
#pragma unroll
    for (int j = 0; j < T::kCopies; ++j) {
        const int row = (wave * T::kCopies + j) * T::kCopyRows + lane / T::kChunks;
        src[j] = T::place(row, chunk_of) * 16;
        off_x[j] = (uint32_t)(min(m0 + row, a.rows - 1) - m0) * (uint32_t)a.xq_stride + src[j];
        int64_t wr;
        if constexpr (GATED) wr = (int64_t)min(n0 + row / 64 * 32 + row % 32, a.n - 1) - n0 + (row & 32 ? a.n : 0);
        else wr = min(n0 + row, a.n - 1) - n0;
        off_w[j] = (uint32_t)(wr * a.w_stride) + src[j];
    }
    const uint8_t* base_x = a.xq + (int64_t)m0 * a.xq_stride;
    const uint8_t* base_w = (const uint8_t*)a.w + (int64_t)n0 * a.w_stride;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const auto copy_x = [&](int step, int j) {
        copy_to_lds(base_x + (int64_t)step * BK, off_x[j],
                    lds0 + (step % S) * 2 * T::kUnit + (wave * T::kCopies + j) * 1024);
    };
    const auto copy_w = [&](int step, int j) {
        // behind the matrix row's last chunk its first of this stage again: the rows hold zeros there
        const uint32_t back = step * BK + src[j] >= kw ? (uint32_t)src[j] : 0u;
        copy_to_lds(base_w + (int64_t)step * BK, off_w[j] - back,
                    lds0 + (step % S) * 2 * T::kUnit + T::kUnit + (wave * T::kCopies + j) * 1024);
    };
    const auto copy_stage = [&](int step) {
#pragma unroll
        for (int j = 0; j < T::kCopies; ++j) {
            copy_x(step, j);
            copy_w(step, j);
        }
    };
    // operands: lane l holds row l % 32, chunk 2 s + l / 32 of step s
    const int wave_m = wave % 2 * (B / 2), wave_n = wave / 2 * (B / 2);
    const int r = lane % 32, half = lane / 32;
    int at_x[T::kSteps], at_w[T::kSteps];
#pragma unroll
    for (int s = 0; s < T::kSteps; ++s) {
        at_x[s] = (wave_m + r) * BK + T::place(r, 2 * s + half) * 16;
        at_w[s] = (wave_n + r) * BK + T::place(r, 2 * s + half) * 16 + T::kUnit;
    }
    v4i xf[2][F], wf[2][F];
    const auto read = [&](int to, int stage, int s) {
        const uint8_t* p = lds + stage * 2 * T::kUnit;
#pragma unroll
        for (int f = 0; f < F; ++f) {
            xf[to][f] = *(const v4i*)(p + at_x[s] + f * 32 * BK);
            wf[to][f] = *(const v4i*)(p + at_w[s] + f * 32 * BK);
        }
    };
    v16i acc[F][F];  // [matrix fragment][row fragment]: lane l holds row l % 32 and matrix rows 8 (i / 4) + 4 (l / 32) + i % 4
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    const auto multiply = [&](int from) {
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) acc[i][j] = mfma_i8_32(wf[from][i], xf[from][j], acc[i][j]);
    };
    for (int s = 0; s < S && s < steps; ++s) copy_stage(s);
    tile_wait<0>();
    read(0, 0, 0);
    for (int t = 0; t < steps; ++t) {
        const int stage = t % S;
#pragma unroll
        for (int s = 0; s < T::kSteps; ++s) {
            if (s + 1 < T::kSteps) {
                read((s + 1) % 2, stage, s + 1);
            } else {
                // every wave has read stage t, and stage t + 1 has come: younger ones may be on their way
                if (t + S - 1 < steps) tile_wait<(S - 2) * 2 * T::kCopies>();
                else tile_wait<0>();
                if (t + S < steps) copy_stage(t + S);
                if (t + 1 < steps) read(0, (t + 1) % S, 0);
            }
            multiply(s % 2);
        }
    }
    // every wave is behind its last read of the ring: each takes a part of it for its results, 32 rows at a time
    constexpr int kWaveCols = GATED ? B / 4 : B / 2, kPitch = kWaveCols + 4;
    static_assert(4 * 32 * kPitch * 4 <= S * 2 * T::kUnit, "results fit the ring");
    float* mine = (float*)lds + wave * 32 * kPitch;
    const int col0 = n0 + wave / 2 * kWaveCols;
#pragma unroll
    for (int j = 0; j < F; ++j) {
        const int row0 = m0 + wave_m + j * 32;
        const float xs = a.xs[min(row0 + r, a.rows - 1)];
        constexpr int kFragments = GATED ? F / 2 : F;
#pragma unroll
        for (int i = 0; i < kFragments; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = i * 32 + q * 8 + half * 4;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = min(col0 + col + e, a.n - 1);
                    if constexpr (GATED) {
                        const float gate = int8_value(acc[2 * i][j][q * 4 + e], a.ws[n], xs);
                        v[e] = int8_gate(gate, a.gelu) * int8_value(acc[2 * i + 1][j][q * 4 + e], a.ws[n + a.n], xs);
                    } else {
                        v[e] = int8_value(acc[i][j][q * 4 + e], a.ws[n], xs);
                    }
                }
                *(v4f*)(mine + r * kPitch + col) = v4f{v[0], v[1], v[2], v[3]};
            }
        constexpr int kVectors = kWaveCols / 8, kRowsAt = kWave / kVectors;
#pragma unroll 1
        for (int p = 0; p < 32 / kRowsAt; ++p) {
            const int rr = p * kRowsAt + lane / kVectors, cc = lane % kVectors * 8, n = col0 + cc;
            const int64_t row = row0 + rr;
            const v4f lo = *(const v4f*)(mine + rr * kPitch + cc), hi = *(const v4f*)(mine + rr * kPitch + cc + 4);
            if (row >= a.rows || n >= a.n) continue;
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (a.bias) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += a.bias[min(n + e, a.n - 1)];
            }
            const auto finish = [&](auto dt) {
                constexpr int DT = decltype(dt)::value;
                if (a.residual) {
                    float add[8];
                    load_cols8<DT>((const char*)a.residual + row * a.residual_stride * elem_bytes<DT>(), n, a.n, add);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += add[e];
                }
                store_cols8<DT>((char*)a.out + row * a.out_stride * elem_bytes<DT>(), n, a.n, v);
            };
            if (a.out_dtype == kBF16) finish(std::integral_constant<int, kBF16>{});
            else if (a.out_dtype == kF16) finish(std::integral_constant<int, kF16>{});
            else finish(std::integral_constant<int, kF32>{});
        }
    }
}

template <int B, int BK, int S>
void launch_tiles_as(const Int8Args& a, hipStream_t stream) {
    const int cols = a.gated ? B / 2 : B;
    const int64_t row_tiles = (a.rows + B - 1) / B, col_tiles = (a.n + cols - 1) / cols;
    const dim3 grid((unsigned)((row_tiles * col_tiles + kTileXcd - 1) / kTileXcd * kTileXcd)), block(256);
    if (a.gated) hipLaunchKernelGGL((int8_tile_kernel<B, BK, S, true>), grid, block, 0, stream, a, (int)row_tiles, (int)col_tiles);
    else hipLaunchKernelGGL((int8_tile_kernel<B, BK, S, false>), grid, block, 0, stream, a, (int)row_tiles, (int)col_tiles);
}

}  // namespace

void launch_int8_tiles(const Int8Args& a, int cus, hipStream_t stream) {
    const int64_t large = (int64_t)((a.rows + 255) / 256) * ((a.n * (a.gated ? 2 : 1) + 255) / 256);
    if (large >= cus) launch_tiles_as<256, 128, 2>(a, stream);
    else launch_tiles_as<128, 128, 2>(a, stream);
}

}  // namespace dmoe
