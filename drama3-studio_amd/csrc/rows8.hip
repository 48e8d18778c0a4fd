// Rows of the residual stream between two blocks of a decoder layer, in one
// pass: the residual's addition, the root-mean-square norm, and the next
// block's input in 8 bits with scales; the row quantizer alone; and what rows
// in 8 bits stand for.
//
//   h = T(x + residual);  g = fl32(offset + weight);  u = fl32(h g)
//   y = u r,  r = 1 / sqrt(sum(h^2) / cols + eps)
//   integers: s = fl32(max(fl32(max|u| r), 1e-12) fl32(1/127)), codes round(u r / s)
//   E4M3:     s = fl32(max(fl32(max|u| r), 1e-10) fl32(1/448)), codes the numbers nearest u r / s
//
// r > 0 is the same for a row, so the row's largest |y| comes from its largest
// |u|: one reduction carries the sum and the maximum, and the row's values
// stay in registers between the two halves.  The sum and r are of 64 bits, so
// that scales and codes are those of the formula and do not depend on how a
// row was cut; the codes are decided in 32 bits except next to a border.
// Memory bounds many rows (8192 of 4096, bf16 with residual to integers: 45 us,
// 5.2 TB/s), a row's latency few (one of 2048: 3.1 us with its launch).
#include <algorithm>

#include "rows8_util.hpp"

namespace dmoe {

namespace {

// Rows of a workgroup of T threads a row: several where a wave holds one.
constexpr int rows_per(int threads) { return threads == kWave ? 4 : 1; }

// T threads hold a row, V vectors of eight columns each.
template <int DT, int T, int V, bool NORM>
__global__ __launch_bounds__(rows_per(T) * T) void rows8_kernel(NormArgs a) {
    constexpr int kRowsPer = rows_per(T);
    constexpr int kWaves = T / kWave;
    constexpr int kBytes = elem_bytes<DT>();
    const int t = threadIdx.x % T;
    const int64_t row = (int64_t)blockIdx.x * kRowsPer + threadIdx.x / T;
    if (row >= a.rows) return;  // whole waves; a row of several waves is a whole workgroup
    const char* x = (const char*)a.x + row * a.x_stride * kBytes;
    Cols8<DT> h[V];
    float u[V][8];
    int top = 0, group_top[V];
    double sum = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = load_raw8<DT>(x, (v * T + t) * 8, a.cols);
    if (NORM && a.residual) {
        const char* r = (const char*)a.residual + row * a.residual_stride * kBytes;
        Cols8<DT> add[V];
#pragma unroll
        for (int v = 0; v < V; ++v) add[v] = load_raw8<DT>(r, (v * T + t) * 8, a.cols);
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[v][j] = col_of<DT>(h[v], j) + col_of<DT>(add[v], j);
            h[v] = cols_of<DT>(u[v]);
        }
        if (a.hidden) {
            char* to = (char*)a.hidden + row * a.hidden_stride * kBytes;
#pragma unroll
            for (int v = 0; v < V; ++v) store_raw8<DT>(to, (v * T + t) * 8, a.cols, h[v]);
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[v][j] = col_of<DT>(h[v], j);
        if constexpr (NORM) {
            float g[8];
            const int col = (v * T + t) * 8;
            if (a.weight_dtype == kBF16) load_cols8<kBF16>(a.weight, col, a.cols, g);
            else if (a.weight_dtype == kF16) load_cols8<kF16>(a.weight, col, a.cols, g);
            else load_cols8<kF32>(a.weight, col, a.cols, g);
            int m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum = __builtin_fma((double)u[v][j], (double)u[v][j], sum);
                u[v][j] *= a.offset + g[j];
                m = max(m, magnitude(u[v][j]));
            }
            group_top[v] = m;
        } else {
            group_top[v] = magnitude8<DT>(h[v]);
        }
        top = max(top, group_top[v]);
    }
    top = wave_max_bits(top);
    if constexpr (NORM) sum = wave_sum_f64(sum);
    if constexpr (kWaves > 1) {
        __shared__ double sums[kWaves];
        __shared__ int tops[kWaves];
        const int wave = t / kWave;
        if (t % kWave == 0) {
            if (NORM) sums[wave] = sum;
            tops[wave] = top;
        }
        __syncthreads();
        sum = NORM ? sums[0] : 0.0;
        top = tops[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            if (NORM) sum += sums[w];
            top = max(top, tops[w]);
        }
    }
    const double by = NORM ? rsqrt_f64(sum / a.cols + a.eps) : 1.0;
    if (NORM && a.y) {
        char* y = (char*)a.y + row * a.y_stride * kBytes;
        const float r = (float)by;
        const bool plain = by > 0x1p-120 && by < 0x1p120;  // elsewhere r is no normal number or soon none
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = plain ? u[v][j] * r : (float)((double)u[v][j] * by);
            store_cols8<DT>(y, (v * T + t) * 8, a.cols, o);
        }
    }
    if (a.q.format == kRowsNone) return;
    uint8_t* q = a.q.q + row * a.q.stride;
    if (a.q.format == kRowsE4M3Group) {  // cols % 128 == 0: sixteen lanes hold a group
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int col = (v * T + t) * 8;
            if (col >= a.cols) continue;
            const float top32 = (float)((double)__int_as_float(row_max_bits(group_top[v])) * by);
            const bool fine = finite_bits(top32);
            const float scale = e4m3_scale(top32);
            *(uint64_t*)(q + col) = fine ? e4m3_codes8(u[v], units_of(by, scale)) : 0;
            if (t % 16 == 0) {
                a.q.scales[row * (a.cols / 128) + col / 128] = fine ? scale : __builtin_nanf("");
                if (!fine) raise_status(a.status, kNonFinite);
            }
        }
        return;
    }
    const float top32 = (float)((double)__int_as_float(top) * by);
    const bool fine = finite_bits(top32), e4m3 = a.q.format == kRowsE4M3;
    const float scale = e4m3 ? e4m3_scale(top32) : int8_scale(top32);
    const Units units = units_of(by, scale);
    const int end = padded_k(a.cols);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int col = (v * T + t) * 8;  // columns from cols on are zeros
        if (col < end)
            *(uint64_t*)(q + col) = !fine ? 0 : e4m3 ? e4m3_codes8(u[v], units) : int8_codes8(u[v], units);
    }
    if (t == 0) {
        a.q.scales[row] = fine ? scale : __builtin_nanf("");
        if (!fine) raise_status(a.status, kNonFinite);
    }
}

// A launch holds fewer than 2^32 threads; more rows take several.
constexpr int kRowsOfLaunch = 1 << 21;

template <int DT, int T, int V>
void launch_rows8_as(NormArgs a, hipStream_t stream) {
    const int per = rows_per(T), all = a.rows;
    const dim3 block(per * T);
    const auto move = [](auto*& p, int64_t bytes) {
        if (p) p = (std::remove_reference_t<decltype(p)>)((char*)p + bytes);
    };
    for (int at = 0;; at += kRowsOfLaunch) {
        a.rows = std::min(all - at, kRowsOfLaunch);
        const dim3 grid((unsigned)((a.rows + per - 1) / per));
        if (a.weight) hipLaunchKernelGGL((rows8_kernel<DT, T, V, true>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((rows8_kernel<DT, T, V, false>), grid, block, 0, stream, a);
        if (all - at <= kRowsOfLaunch) return;
        constexpr int64_t kMoved = (int64_t)kRowsOfLaunch * elem_bytes<DT>();
        move(a.x, a.x_stride * kMoved);
        move(a.residual, a.residual_stride * kMoved);
        move(a.hidden, a.hidden_stride * kMoved);
        move(a.y, a.y_stride * kMoved);
        move(a.q.q, a.q.stride * kRowsOfLaunch);
        move(a.q.scales, (a.q.format == kRowsE4M3Group ? a.cols / 128 : 1) * (int64_t)kRowsOfLaunch * 4);
    }
}

// Two vectors a thread: its loads are on their way together, and a row's fixed part (sums of 64 bits, factors) is shared
// by few threads.  Norms with residual, bf16, us: 8192 rows of 2048 by 128 threads 26.0, by 256 with one vector 36.2; 4000
// rows of 1024 by 64 threads 9.1, with four vectors 10.3; 300 rows of 8192 by 512 threads 7.6, by 1024 with one 11.4, by
// 256 with four 8.2; 2000 rows of 5120 by 256 threads with three 19.4, by 512 with two 20.5 (13.1 and 16.8 out of the
// caches).  Rows that do not fill the chip get more threads each, or less code: their time is a row's (one row of 2048 to
// E4M3 groups by 256 threads with one vector 3.4, with two 4.2; 250 rows of 2048 by 256 threads 4.2, by 128 4.6; 47 rows
// of 14336 by 1024 threads 5.9, by 512 with four vectors 6.4, and 2000 such rows 43.4, 40.4).  E4M3 groups have nothing
// that two vectors share (400 rows of 2048 by 256 threads with one 4.4, by 128 5.5; 2000 8.9 and 8.5).  Eight vectors a
// thread, above 32768 columns, spill: 24 registers in norms of 16-bit types, 82 in the quantizer of fp16, 125 in the norm
// of fp32 (2000 rows of 33024 and of 32768: 104 and 77, 52 and 46, 318 and 127).
template <int DT>
void launch_rows8_of(const NormArgs& a, hipStream_t stream) {
    const int end = padded_k(a.cols);
    const bool few = a.rows <= 256;
    if (end <= 1024) return launch_rows8_as<DT, 64, 2>(a, stream);
    const bool groups = a.q.format == kRowsE4M3Group && a.rows <= 1024;
    if (end <= 2048) return few || groups ? launch_rows8_as<DT, 256, 1>(a, stream) : launch_rows8_as<DT, 128, 2>(a, stream);
    if (end <= 4096) return launch_rows8_as<DT, 256, 2>(a, stream);
    if (end <= 6144 && !few) return launch_rows8_as<DT, 256, 3>(a, stream);
    if (end <= 8192) return launch_rows8_as<DT, 512, 2>(a, stream);
    if (end <= 12288 && !few) return launch_rows8_as<DT, 512, 3>(a, stream);
    if (end <= 16384) return few ? launch_rows8_as<DT, 1024, 2>(a, stream) : launch_rows8_as<DT, 512, 4>(a, stream);
    if (end <= 32768) return launch_rows8_as<DT, 1024, 4>(a, stream);
    return launch_rows8_as<DT, 1024, 8>(a, stream);
}

template <int DT>
__global__ __launch_bounds__(256) void dequant8_kernel(Dequant8Args a, int per_row, int64_t first, int64_t total) {
    const int64_t i = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t row = i / per_row;
    const int col = (int)(i - row * per_row) * 8;
    const uint8_t* q = a.q.q + row * a.q.stride + col;
    const float scale = a.q.scales[a.q.format == kRowsE4M3Group ? row * (a.cols / 128) + col / 128 : row];
    float v[8];
    const uint64_t w = *(const uint64_t*)q;  // rows are readable to a multiple of sixteen columns
    if (a.q.format == kRowsInt8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)(int8_t)(w >> (8 * j)) * scale;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const v2f two = fp8x2_to_f32((uint32_t)(j < 2 ? w : w >> 32), j % 2 != 0);
            v[2 * j] = two[0] * scale;
            v[2 * j + 1] = two[1] * scale;
        }
    }
    store_cols8<DT>((char*)a.out + row * a.out_stride * elem_bytes<DT>(), col, a.cols, v);
}

}  // namespace

void launch_rows8(const NormArgs& a, hipStream_t stream) {
    if (a.dtype == kBF16) launch_rows8_of<kBF16>(a, stream);
    else if (a.dtype == kF16) launch_rows8_of<kF16>(a, stream);
    else launch_rows8_of<kF32>(a, stream);
}

void launch_dequant8(const Dequant8Args& a, hipStream_t stream) {
    const int per_row = (a.cols + 7) / 8;
    const int64_t total = (int64_t)a.rows * per_row;
    constexpr int64_t kLaunch = (int64_t)1 << 31;  // threads: fewer than 2^32
    for (int64_t first = 0; first < total; first += kLaunch) {
        const dim3 grid((unsigned)((std::min(total - first, kLaunch) + 255) / 256)), block(256);
        const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a, per_row, first, total); };
        if (a.dtype == kBF16) go(dequant8_kernel<kBF16>);
        else if (a.dtype == kF16) go(dequant8_kernel<kF16>);
        else go(dequant8_kernel<kF32>);
    }
}

}  // namespace dmoe
