// Argument blocks and launchers of rows and products in 8 bits: the norm with
// the residual's addition, the row quantizers (rows8.hip), and the products of
// 8-bit integer rows and matrices (int8_few.hip, int8_tiles.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dmoe {

constexpr int kInt8MaxK = 65536;      // 2^16 products of at most 2^14: an int32 sum holds them
constexpr int kRows8MaxRows = 1 << 24;
constexpr int kInt8Pad = 128;         // quantized rows hold zeros up to a multiple of this many columns

// What rows leave as in 8 bits.
enum Rows8Format : int { kRowsNone = 0, kRowsInt8 = 1, kRowsE4M3 = 2, kRowsE4M3Group = 3 };

__host__ __device__ inline int padded_k(int k) { return (k + kInt8Pad - 1) / kInt8Pad * kInt8Pad; }

// Rows [rows, cols] of a float type; a stride in elements.
struct Rows {
    void* p = nullptr;
    int64_t stride = 0;
    int dtype = 0;
};

// Rows in 8 bits with their scales ([rows], or [rows, cols / 128]); a stride in bytes.
struct Rows8 {
    uint8_t* q = nullptr;
    int64_t stride = 0;
    float* scales = nullptr;
    int format = kRowsNone;
};

struct NormArgs {
    const void* x;
    int64_t x_stride;
    const void* residual;  // may be null
    int64_t residual_stride;
    int dtype;             // of x, residual, hidden and y
    int rows, cols;
    const void* weight;    // null: rows are quantized as they are, without a norm
    int weight_dtype;
    float offset;
    double eps;
    void* hidden;          // x + residual; may be null
    int64_t hidden_stride;
    void* y;               // may be null
    int64_t y_stride;
    Rows8 q;               // format kRowsNone: not wanted
    int* status;
};

struct Dequant8Args {
    Rows8 q;
    int rows, cols;
    void* out;
    int64_t out_stride;
    int dtype;
};

// out = act(x w^T): w [n, k] (gated: [2 n, k], gate rows first) of 8-bit integers.
struct Int8Args {
    // activation rows: quantized (xq, zeros in [k, padded_k(k))), or of a float type (x) for the kernel to quantize
    const uint8_t* xq;
    int64_t xq_stride;
    const float* xs;
    const void* x;
    int64_t x_stride;
    int x_dtype;
    int rows, k;
    const int8_t* w;
    int64_t w_stride;
    const float* ws;
    int n;                 // output columns
    int gated, gelu;       // out = act(gate) * up
    const float* bias;     // may be null
    const void* residual;  // of out's type; may be null
    int64_t residual_stride;
    void* out;
    int64_t out_stride;
    int out_dtype;
    int* status;
};

void launch_rows8(const NormArgs& a, hipStream_t stream);
void launch_dequant8(const Dequant8Args& a, hipStream_t stream);

constexpr int kInt8FewRows = 64;    // rows that the kernel of few rows takes
// Whether that kernel quantizes `rows` rows of k columns itself.
bool int8_few_quantizes(int rows, int k);
void launch_int8_few(const Int8Args& a, hipStream_t stream);
void launch_int8_tiles(const Int8Args& a, int cus, hipStream_t stream);

}  // namespace dmoe
