// Products of few rows of 8-bit integers with a matrix of them.
//
//   acc[t][n] = sum_k xq[t][k] w[n][k] (int32, exact), out = T(acc xs[t] ws[n] + bias[n] + residual[t][n]),
//   gated: out = T(act(gate) up) of the products with rows n and n + N of w
//
// The matrix is read once and bounds the call.  A workgroup owns NT tiles of
// sixteen matrix rows; its waves cut K into blocks of 128 columns, each lane
// streaming 16-byte pieces of one row into 16x16x64 matrix instructions, and
// add their sums in LDS: integer sums, so their order does not matter.  Up to
// four rows that are not quantized yet are quantized by every workgroup for
// itself while its first matrix pieces are on their way (a row is at most
// 64 KB from L2, less than a launch of its own costs).
#include <algorithm>

#include "rows8_util.hpp"
#include "int8_epilogue.hpp"

namespace dmoe {

namespace {

constexpr int kFewWaves = 8;
constexpr int kFewBlock = 128;      // columns of a K block
constexpr int kFewSumPitch = 17;    // ints from one row's sums to the next row's: 16 and one against bank conflicts
constexpr int kFewQuantRows = 4, kFewQuantVectors = 4;
constexpr int kFewQuantBytes = 32768;

template <int DT>
__device__ __forceinline__ void quantize_to_lds(const Int8Args& a, uint8_t* lds, int pitch, float* lds_scale, int* tops) {
    const int waves = kFewWaves;
    const int slots = a.rows == 1 ? 1 : a.rows == 2 ? 2 : 4;  // wave groups, one a row
    const int per = waves / slots, threads = per * kWave;
    const int wave = threadIdx.x / kWave, group = wave / per, t = threadIdx.x - group * threads;
    const int row = min(group, a.rows - 1), end = padded_k(a.k);
    const char* x = (const char*)a.x + (int64_t)row * a.x_stride * elem_bytes<DT>();
    float u[kFewQuantVectors][8];
    int top = 0;
#pragma unroll
    for (int v = 0; v < kFewQuantVectors; ++v) {
        load_cols8<DT>(x, (v * threads + t) * 8, a.k, u[v]);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude(u[v][j]));
    }
    top = wave_max_bits(top);
    if (threadIdx.x % kWave == 0) tops[wave] = top;
    lds_barrier();
    top = tops[group * per];
    for (int w = 1; w < per; ++w) top = max(top, tops[group * per + w]);
    const float top32 = __int_as_float(top);
    const bool fine = finite_bits(top32);
    const float scale = int8_scale(top32), each = __fdiv_rn(1.0f, scale);
    if (group < a.rows) {
#pragma unroll
        for (int v = 0; v < kFewQuantVectors; ++v) {
            const int col = (v * threads + t) * 8;
            if (col < end) *(uint64_t*)(lds + row * pitch + col) = fine ? int8_codes8(u[v], each, 1.0, scale) : 0;
        }
        if (t == 0) {
            lds_scale[row] = fine ? scale : __builtin_nanf("");
            if (!fine && blockIdx.x == 0) raise_status(a.status, kNonFinite);
        }
    }
    lds_barrier();
}

// U K blocks of a wave are in flight at a time.
template <int NT, int MT, bool GATED, bool QUANT>
__global__ __launch_bounds__(kFewWaves * kWave) void int8_few_kernel(Int8Args a) {
    constexpr int kCols = GATED ? NT * 8 : NT * 16;
    constexpr int U = NT * MT >= 8 ? 1 : NT >= 4 ? 2 : 4;
    __shared__ int sums[NT * MT * 16 * kFewSumPitch];
    __shared__ alignas(16) uint8_t xl[QUANT ? kFewQuantBytes : 16];
    __shared__ float xl_scale[QUANT ? kFewQuantRows : 1];
    __shared__ int tops[QUANT ? kFewWaves : 1];
    const int lane = threadIdx.x % kWave, r = lane % 16, c = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), waves = kFewWaves;
    const int n0 = blockIdx.x * kCols;
    const int blocks = (a.k + kFewBlock - 1) / kFewBlock;
    const int last = ((a.k + 15) / 16 - 1) * 16;  // the last piece of a matrix row; rows' zeros stand against what repeats
    const uint8_t* wrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int col = min(n0 + (GATED ? j % (NT / 2) : j) * 16 + r, a.n - 1);
        wrow[j] = (const uint8_t*)a.w + (int64_t)(GATED && j >= NT / 2 ? col + a.n : col) * a.w_stride;
    }
    v4i wf[U][NT][2];
    const auto fetch = [&](int b0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(b0 + u * waves, blocks - 1) * kFewBlock + c * 16;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) wf[u][j][h] = *(const v4i*)(wrow[j] + min(at + h * 64, last));
        }
    };
    fetch(wave);
    for (int i = threadIdx.x; i < NT * MT * 16 * kFewSumPitch; i += kFewWaves * kWave) sums[i] = 0;
    const int pitch = padded_k(a.k) + 16;
    if constexpr (QUANT) {
        if (a.x_dtype == kBF16) quantize_to_lds<kBF16>(a, xl, pitch, xl_scale, tops);
        else if (a.x_dtype == kF16) quantize_to_lds<kF16>(a, xl, pitch, xl_scale, tops);
        else quantize_to_lds<kF32>(a, xl, pitch, xl_scale, tops);
    } else {
        lds_barrier();
    }
    v4i acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[j][m] = v4i{0, 0, 0, 0};
    const v4i zero = {0, 0, 0, 0};
    for (int b0 = wave; b0 < blocks; b0 += U * waves) {
        if (b0 != wave) fetch(b0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + u * waves;
            if (b < blocks) {
                const int at = b * kFewBlock + c * 16;
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const int row = m * 16 + r;
                    v4i xf[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if constexpr (QUANT) xf[h] = row < a.rows ? *(const v4i*)(xl + row * pitch + at + h * 64) : zero;
                        else xf[h] = row < a.rows ? *(const v4i*)(a.xq + (int64_t)row * a.xq_stride + at + h * 64) : zero;
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) acc[j][m] = mfma_i8(wf[u][j][h], xf[h], acc[j][m]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) atomicAdd(&sums[((j * MT + m) * 16 + r) * kFewSumPitch + 4 * c + i], acc[j][m][i]);
    lds_barrier();
    for (int i = threadIdx.x; i < MT * 16 * kCols; i += kFewWaves * kWave) {
        const int row = i / kCols, col = i % kCols, n = n0 + col;
        if (row >= a.rows || n >= a.n) continue;
        const int j = col / 16, m = row / 16;
        const float xs = QUANT ? xl_scale[QUANT ? row : 0] : a.xs[row];
        const int* s = &sums[((j * MT + m) * 16 + row % 16) * kFewSumPitch + col % 16];
        float v = int8_value(s[0], a.ws[n], xs);
        if constexpr (GATED)
            v = int8_gate(v, a.gelu) * int8_value(s[NT / 2 * MT * 16 * kFewSumPitch], a.ws[n + a.n], xs);
        if (a.bias) v += a.bias[n];
        if (a.residual) v += load_as_f32(a.residual, (int64_t)row * a.residual_stride + n, a.out_dtype);
        store_from_f32(a.out, (int64_t)row * a.out_stride + n, a.out_dtype, v);
    }
}

template <int NT, int MT, bool GATED>
void launch_few_as(const Int8Args& a, hipStream_t stream) {
    constexpr int kCols = GATED ? NT * 8 : NT * 16;
    const dim3 grid((unsigned)((a.n + kCols - 1) / kCols)), block(kFewWaves * kWave);
    if constexpr (MT == 1) {
        if (a.xq == nullptr) {
            hipLaunchKernelGGL((int8_few_kernel<NT, MT, GATED, true>), grid, block, 0, stream, a);
            return;
        }
    }
    hipLaunchKernelGGL((int8_few_kernel<NT, MT, GATED, false>), grid, block, 0, stream, a);
}

template <int NT, bool GATED>
void launch_few_of(const Int8Args& a, hipStream_t stream) {
    if (a.rows <= 16) launch_few_as<NT, 1, GATED>(a, stream);
    else if (a.rows <= 32) launch_few_as<NT, 2, GATED>(a, stream);
    else launch_few_as<NT, 4, GATED>(a, stream);
}

}  // namespace

bool int8_few_quantizes(int rows, int k) {
    if (rows > kFewQuantRows || rows * (padded_k(k) + 16) > kFewQuantBytes) return false;
    const int slots = rows == 1 ? 1 : rows == 2 ? 2 : 4;
    return padded_k(k) <= kFewQuantVectors * 8 * (kFewWaves / slots) * kWave;
}

void launch_int8_few(const Int8Args& a, hipStream_t stream) {
    if (a.gated) launch_few_of<2, true>(a, stream);
    else launch_few_of<1, false>(a, stream);
}

}  // namespace dmoe
