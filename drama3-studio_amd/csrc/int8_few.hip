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
// itself while its first matrix pieces are on their way (one row, K 2048, N
// 2560: 3.6 us against 3.3 and a launch of the quantizer, about 2.5).
#include "rows8_util.hpp"
#include "int8_epilogue.hpp"

namespace dmoe {

namespace {

constexpr int kFewBlock = 128;      // columns of a K block
constexpr int kFewSumPitch = 17;    // ints from one row's sums to the next row's: 16 and one against bank conflicts
constexpr int kFewQuantRows = 4;
constexpr int kFewQuantBytes = 32768;

// The call's rows to 8-bit integers in LDS, a row by each group of waves.  A
// thread holds its first eight columns, asked for before the matrix's loads
// (they would be waited for too); longer rows are read twice rather than
// held, which would cost those loads their registers.
template <int DT, int W>
struct RowsToLds {
    int group, t, threads, row;
    const char* x;
    Cols8<DT> first;

    __device__ __forceinline__ RowsToLds(const Int8Args& a, bool wanted) {
        if (!wanted) return;
        const int slots = a.rows == 1 ? 1 : a.rows == 2 ? 2 : 4;
        threads = W / slots * kWave;
        group = threadIdx.x / threads;
        t = threadIdx.x - group * threads;
        row = min(group, a.rows - 1);
        x = (const char*)a.x + (int64_t)row * a.x_stride * elem_bytes<DT>();
        first = load_raw8<DT>(x, t * 8, a.k);
    }

    __device__ __forceinline__ void quantize(const Int8Args& a, uint8_t* lds, int pitch, float* lds_scale, int* tops) const {
        const int per = threads / kWave, end = padded_k(a.k);
        int top = magnitude8<DT>(first);
#pragma unroll 1
        for (int col = (t + threads) * 8; col < a.k; col += threads * 8) top = max(top, magnitude8<DT>(load_raw8<DT>(x, col, a.k)));
        top = wave_max_bits(top);
        if (threadIdx.x % kWave == 0) tops[threadIdx.x / kWave] = top;
        lds_barrier();
        top = tops[group * per];
        for (int w = 1; w < per; ++w) top = max(top, tops[group * per + w]);
        const float top32 = __int_as_float(top);
        const bool fine = finite_bits(top32);
        const Units units = units_of(1.0, int8_scale(top32));
        if (group < a.rows) {
            Cols8<DT> c = first;
#pragma unroll 1
            for (int col = t * 8; col < end; col += threads * 8) {
                if (col != t * 8) c = load_raw8<DT>(x, col, a.k);
                float u[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] = col_of<DT>(c, j);
                *(uint64_t*)(lds + row * pitch + col) = fine ? int8_codes8(u, units) : 0;
            }
            if (t == 0) {
                lds_scale[row] = fine ? units.scale : __builtin_nanf("");
                if (!fine && blockIdx.x == 0) raise_status(a.status, kNonFinite);
            }
        }
        lds_barrier();
    }
};

// A wave's next block is on its way while it multiplies one.
// DT is the type of rows that are not quantized yet, kI32 where they are.
template <int NT, int MT, int W, bool GATED, int DT>
__global__ __launch_bounds__(W * kWave, (W > 8 ? 4 : NT * MT <= 2 ? 6 : NT * MT <= 4 ? 4 : 2)) void int8_few_kernel(Int8Args a) {
    constexpr bool QUANT = DT != kI32;
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
        v4i w[NT][2], x[QUANT ? 1 : MT][2];
    };
    const auto fetch = [&](Group& g, int b) {
        const int at = min(b, blocks - 1) * kFewBlock + c * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NT; ++j) g.w[j][h] = *(const v4i*)(wrow[j] + min(at + h * 64, last));
            if constexpr (!QUANT) {
#pragma unroll
                for (int m = 0; m < MT; ++m) g.x[m][h] = *(const v4i*)(xrow[m] + at + h * 64);
            }
        }
    };
    const RowsToLds<QUANT ? DT : kBF16, W> rows(a, QUANT);
    Group now, next;
    fetch(now, wave);
    // what the first result of a thread needs beside its sum
    const int my_row = threadIdx.x / kCols, my_n = min(n0 + (int)threadIdx.x % kCols, a.n - 1);
    const int safe_row = min(my_row, a.rows - 1);
    const float my_ws = a.ws[my_n], my_up = GATED ? a.ws[my_n + a.n] : 0.0f, my_xs = QUANT ? 0.0f : a.xs[safe_row];
    const float my_bias = a.bias ? a.bias[my_n] : 0.0f;
    const float my_add = a.residual ? load_as_f32(a.residual, (int64_t)safe_row * a.residual_stride + my_n, a.out_dtype) : 0.0f;
    for (int i = threadIdx.x; i < NT * MT * 16 * kFewSumPitch; i += W * kWave) sums[i] = 0;
    if constexpr (QUANT) rows.quantize(a, xl, pitch, xl_scale, tops);
    else lds_barrier();
    v4i acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[j][m] = v4i{0, 0, 0, 0};
    const auto multiply = [&](const Group& g, int b) {
        if (b >= blocks) return;  // the same for the wave
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4i xf = QUANT ? *(const v4i*)(xlds + b * kFewBlock + c * 16 + h * 64) : g.x[QUANT ? 0 : m][h];
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][m] = mfma_i8(g.w[j][h], xf, acc[j][m]);
            }
    };
    int b = wave;
    while (true) {
        const bool more = b + W < blocks;
        if (more) fetch(next, b + W);
        multiply(now, b);
        if (!more) break;
        b += W;
        const bool again = b + W < blocks;
        if (again) fetch(now, b + W);
        multiply(next, b);
        if (!again) break;
        b += W;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) atomicAdd(&sums[((j * MT + m) * 16 + r) * kFewSumPitch + 4 * c + i], acc[j][m][i]);
    lds_barrier();
    const auto finish = [&](int row, int col, float ws, float up, float xs, float bias, float add) {
        const int j = col / 16, m = row / 16, n = n0 + col;
        const int* s = &sums[((j * MT + m) * 16 + row % 16) * kFewSumPitch + col % 16];
        float v = int8_value(s[0], ws, xs);
        if constexpr (GATED) v = int8_gate(v, a.gelu) * int8_value(s[NT / 2 * MT * 16 * kFewSumPitch], up, xs);
        if (a.bias) v += bias;
        if (a.residual) v += add;
        store_from_f32(a.out, (int64_t)row * a.out_stride + n, a.out_dtype, v);
    };
    if (my_row < min(a.rows, MT * 16) && n0 + (int)threadIdx.x % kCols < a.n)
        finish(my_row, threadIdx.x % kCols, my_ws, my_up, QUANT ? xl_scale[QUANT ? my_row : 0] : my_xs, my_bias, my_add);
    for (int i = threadIdx.x + W * kWave; i < min(a.rows, MT * 16) * kCols; i += W * kWave) {
        const int row = i / kCols, col = i % kCols, n = n0 + col;
        if (n >= a.n) continue;
        finish(row, col, a.ws[n], GATED ? a.ws[n + a.n] : 0.0f, QUANT ? xl_scale[QUANT ? row : 0] : a.xs[row],
               a.bias ? a.bias[n] : 0.0f,
               a.residual ? load_as_f32(a.residual, (int64_t)row * a.residual_stride + n, a.out_dtype) : 0.0f);
    }
}

template <int NT, int MT, int W, bool GATED, int DT>
void launch_few_as(const Int8Args& a, hipStream_t stream) {
    constexpr int kCols = GATED ? NT * 8 : NT * 16;
    hipLaunchKernelGGL((int8_few_kernel<NT, MT, W, GATED, DT>), dim3((unsigned)((a.n + kCols - 1) / kCols)), dim3(W * kWave), 0,
                       stream, a);
}

// Rows of a float type, which the workgroups quantize.
template <int NT, int W, bool GATED>
void launch_few_floats(const Int8Args& a, hipStream_t stream) {
    if (a.x_dtype == kBF16) launch_few_as<NT, 1, W, GATED, kBF16>(a, stream);
    else if (a.x_dtype == kF16) launch_few_as<NT, 1, W, GATED, kF16>(a, stream);
    else launch_few_as<NT, 1, W, GATED, kF32>(a, stream);
}

}  // namespace

bool int8_few_quantizes(int rows, int k) {
    return rows <= kFewQuantRows && rows * (padded_k(k) + 16) <= kFewQuantBytes;
}

// Eight waves a workgroup, or sixteen: those have a K block each from K 2048 on and one round of workgroups to 256 (us,
// eight in brackets; one row of floats, N 2048: K 1024 3.4 (3.1), 1280 3.6 (3.5), 1536 3.6 (3.6), 1792 3.7 (3.7), 2048 3.5
// (3.8); K 5632: N 1280 5.6 (6.2), 4096 7.0 (8.3), 5120 11.1 (10.3)).  In between they are faster where the workgroups
// quantize rows, which goes by threads (four rows, K 5632, N 2048: 8.1 (9.1)); where up to eight rows leave the call to the
// matrix (four, K 5632: N 2048 6.1 (6.4), 4096 6.5 (7.1); eight, K 11008, N 2048 10.9 (10.9)); and where more than 32 rows
// take the registers of all but two waves a SIMD (48 rows, K 4096: N 2048 9.7 (10.3), 4096 10.4 (11.1)).  Not for those
// between (13 rows, K 11008, N 2048 12.2 (11.5); 32 rows, K 2048, N 2560 5.0 (4.9)).  A second K block on its way costs the
// registers of a workgroup a CU (13 rows, K 4096, N 4096: 8.0 us against 6.6).
void launch_int8_few(const Int8Args& a, hipStream_t stream) {
    constexpr int kCus = 256, kWide = 1536;
    const bool sixteen = a.k > kWide && a.n <= 16 * kCus;
    if (a.xq == nullptr) {
        if (a.gated) launch_few_floats<2, 8, true>(a, stream);
        else if (sixteen) launch_few_floats<1, 16, false>(a, stream);
        else launch_few_floats<1, 8, false>(a, stream);
    } else if (a.rows <= 16) {
        if (a.gated) launch_few_as<2, 1, 8, true, kI32>(a, stream);
        else if (sixteen && a.rows <= 8) launch_few_as<1, 1, 16, false, kI32>(a, stream);
        else launch_few_as<1, 1, 8, false, kI32>(a, stream);
    } else if (a.rows <= 32) {
        if (a.gated) launch_few_as<2, 2, 8, true, kI32>(a, stream);
        else launch_few_as<1, 2, 8, false, kI32>(a, stream);
    } else {
        if (a.gated) launch_few_as<2, 4, 8, true, kI32>(a, stream);
        else if (sixteen) launch_few_as<1, 4, 16, false, kI32>(a, stream);
        else launch_few_as<1, 4, 8, false, kI32>(a, stream);
    }
}

}  // namespace dmoe
