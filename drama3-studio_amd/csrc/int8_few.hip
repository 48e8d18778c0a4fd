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

template <int DT, int W>
__device__ __forceinline__ void quantize_to_lds(const Int8Args& a, uint8_t* lds, int pitch, float* lds_scale, int* tops) {
    const int waves = W;
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

// A wave's next U blocks are on their way while it multiplies U.
template <int NT, int MT, int U, int W, bool GATED, bool QUANT>
__global__ __launch_bounds__(W * kWave) void int8_few_kernel(Int8Args a) {
    constexpr int kCols = GATED ? NT * 8 : NT * 16;
    __shared__ int sums[NT * MT * 16 * kFewSumPitch];
    __shared__ alignas(16) uint8_t xl[QUANT ? kFewQuantBytes : 16];
    __shared__ float xl_scale[QUANT ? kFewQuantRows : 1];
    __shared__ int tops[QUANT ? W : 1];
    const int lane = threadIdx.x % kWave, r = lane % 16, c = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n0 = blockIdx.x * kCols;
    const int blocks = (a.k + kFewBlock - 1) / kFewBlock;
    const int last = ((a.k + 15) / 16 - 1) * 16;  // the last piece of a matrix row; rows' zeros stand against what repeats
    const uint8_t* wrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int col = min(n0 + (GATED ? j % (NT / 2) : j) * 16 + r, a.n - 1);
        wrow[j] = (const uint8_t*)a.w + (int64_t)(GATED && j >= NT / 2 ? col + a.n : col) * a.w_stride;
    }
    // a lane beyond the rows reads the last one again: its sums are columns of their own, which nothing takes
    const uint8_t* xrow[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xrow[m] = QUANT ? nullptr : a.xq + (int64_t)min(m * 16 + r, a.rows - 1) * a.xq_stride;
    const int pitch = padded_k(a.k) + 16;
    const uint8_t* xlds = xl + (QUANT ? min(r, a.rows - 1) * pitch : 0);
    struct Group {
        v4i w[U][NT][2], x[QUANT ? 1 : U][QUANT ? 1 : MT][2];
    };
    const auto fetch = [&](Group& g, int b0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(b0 + u * W, blocks - 1) * kFewBlock + c * 16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int j = 0; j < NT; ++j) g.w[u][j][h] = *(const v4i*)(wrow[j] + min(at + h * 64, last));
                if constexpr (!QUANT) {
#pragma unroll
                    for (int m = 0; m < MT; ++m) g.x[u][m][h] = *(const v4i*)(xrow[m] + at + h * 64);
                }
            }
        }
    };
    Group now, next;
    fetch(now, wave);
    for (int i = threadIdx.x; i < NT * MT * 16 * kFewSumPitch; i += W * kWave) sums[i] = 0;
    if constexpr (QUANT) {
        if (a.x_dtype == kBF16) quantize_to_lds<kBF16, W>(a, xl, pitch, xl_scale, tops);
        else if (a.x_dtype == kF16) quantize_to_lds<kF16, W>(a, xl, pitch, xl_scale, tops);
        else quantize_to_lds<kF32, W>(a, xl, pitch, xl_scale, tops);
    } else {
        lds_barrier();
    }
    v4i acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[j][m] = v4i{0, 0, 0, 0};
    const auto multiply = [&](const Group& g, int b0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + u * W;
            if (b >= blocks) continue;  // the same for the wave
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const v4i xf = QUANT ? *(const v4i*)(xlds + b * kFewBlock + c * 16 + h * 64) : g.x[QUANT ? 0 : u][QUANT ? 0 : m][h];
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[j][m] = mfma_i8(g.w[u][j][h], xf, acc[j][m]);
                }
        }
    };
    int b0 = wave;
    while (true) {
        const bool more = b0 + U * W < blocks;
        if (more) fetch(next, b0 + U * W);
        multiply(now, b0);
        if (!more) break;
        b0 += U * W;
        const bool again = b0 + U * W < blocks;
        if (again) fetch(now, b0 + U * W);
        multiply(next, b0);
        if (!again) break;
        b0 += U * W;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) atomicAdd(&sums[((j * MT + m) * 16 + r) * kFewSumPitch + 4 * c + i], acc[j][m][i]);
    lds_barrier();
    for (int i = threadIdx.x; i < MT * 16 * kCols; i += W * kWave) {
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

template <int NT, int MT, int U, int W, bool GATED>
void launch_few_as(const Int8Args& a, hipStream_t stream) {
    constexpr int kCols = GATED ? NT * 8 : NT * 16;
    const dim3 grid((unsigned)((a.n + kCols - 1) / kCols)), block(W * kWave);
    if constexpr (MT == 1) {
        if (a.xq == nullptr) {
            hipLaunchKernelGGL((int8_few_kernel<NT, MT, U, W, GATED, true>), grid, block, 0, stream, a);
            return;
        }
    }
    hipLaunchKernelGGL((int8_few_kernel<NT, MT, U, W, GATED, false>), grid, block, 0, stream, a);
}

template <int NT, bool GATED>
void launch_few_of(const Int8Args& a, hipStream_t stream) {
    if (a.rows <= 16) launch_few_as<NT, 1, 2, kFewWaves, GATED>(a, stream);
    else if (a.rows <= 32) launch_few_as<NT, 2, 1, kFewWaves, GATED>(a, stream);
    else launch_few_as<NT, 4, 1, kFewWaves, GATED>(a, stream);
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
