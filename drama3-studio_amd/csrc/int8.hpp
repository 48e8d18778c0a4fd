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
    int splits;            // shares of K whose sums meet in `part` [splits, rows, int8_part_cols]
    int* part;
    int* status;
};

// Columns of a share's row of sums: whole pieces of eight, gate and up behind each other.
__host__ __device__ inline int64_t int8_part_cols(int n, bool gated) { return (int64_t)((n + 7) / 8 * 8) * (gated ? 2 : 1); }

void launch_rows8(const NormArgs& a, hipStream_t stream);
void launch_dequant8(const Dequant8Args& a, hipStream_t stream);

// How a product is cut.
enum Int8Shape : int { kInt8Few, kInt8Tiles64, kInt8Tiles64x128, kInt8Tiles128Deep, kInt8Tiles128x256, kInt8Tiles128, kInt8Tiles256 };
constexpr int kInt8MaxSplits = 4;
struct Int8Plan {
    Int8Shape shape;
    int splits;  // shares of K, tiles of 64 x 64 only
};

constexpr int kInt8FewRows = 64;  // rows that the kernel of few rows takes

// Every result is the same bits whichever is taken.  A CU brings at most 50 GB/s from memory, 35 (2.2 TB/s) where 64 of
// them do and 18 (4.7 TB/s) where all do, whatever is on its way, and 140 GB/s from L2: a matrix is read fast only by
// most of them, and tiles' rings deeper than three steps or operands read a whole step ahead gain nothing (47 rows, K
// 4096, gated N 11008: 24.4 with three to six steps).  Measured on MI355X (256 CUs) with matrices that are in no cache, us:
// * Few rows: each workgroup of sixteen columns reads all rows, from L2.  Up to 72 MB of that it is as fast as tiles or
//   faster (13 rows, K 4096, N 4096: 6.6 against 13.5; 64 rows, 67 MB: 11.8 against 13.6), above it slower (47 rows,
//   132 MB: K 4096, gated N 11008 39 against 24; K 11008, N 4096 25 against 16.5).
// * 64 x 64 while they do not outnumber the CUs (256 rows, K 4096, N 4096, 256 tiles: 13.8, 64 x 128 17.4, 128 x 128
//   22.5).  A step along K takes about 0.3, so where there are over twenty a share, up to four workgroups share a tile
//   (47 rows, K 11008, N 4096: 28.4 in one, 20.8 in two, 16.5 in four); with fewer, joining costs what it saves (128
//   rows, K 4096, N 4096: 13.6, 14.3, 16.7).
// * 64 x 128 while they do not (47 rows, K 4096, gated N 11008, 172 tiles: 24.2, 64 x 64 26.2, 128 x 128 26.5).
// * 128 x 128 with a deep ring while they do not (509 rows, K 2048, N 5003, 160 tiles: 14.6, 64 x 128 19.5).
// * 128 x 256 while they do not (2048 rows, K 4096, N 4096, 256 tiles: 36.3, 128 x 128 41.9, 256 x 256 52.7).
// * 256 x 256 where their rounds take less than those of 128 x 128 with a ring of two stages, two workgroups a CU: one
//   a CU takes as long as 1 / 0.64 rounds of the others (8192 rows, K 4096, N 4096: 122 against 146).
inline Int8Plan int8_plan(int rows, int n, int k, bool gated) {
    constexpr int64_t kCus = 256;
    const auto tiles = [&](int tm, int tn) {
        const int cols = gated ? tn / 2 : tn;
        return ((int64_t)rows + tm - 1) / tm * (((int64_t)n + cols - 1) / cols);
    };
    const int64_t again = ((int64_t)n + 15) / 16 * rows * k;
    if (rows <= kInt8FewRows && again <= 72000000) return {kInt8Few, 1};
    const int64_t small = tiles(64, 64), middle = tiles(128, 128), large = tiles(256, 256);
    if (small <= kCus) {
        const int64_t steps = (k + 127) / 128, most = kCus / small < steps / 20 ? kCus / small : steps / 20;
        return {kInt8Tiles64, most < 1 ? 1 : most > kInt8MaxSplits ? kInt8MaxSplits : (int)most};
    }
    if (tiles(64, 128) <= kCus) return {kInt8Tiles64x128, 1};
    if (middle <= kCus) return {kInt8Tiles128Deep, 1};
    if (tiles(128, 256) <= kCus) return {kInt8Tiles128x256, 1};
    if ((large + kCus - 1) / kCus * 100 <= (middle + 2 * kCus - 1) / (2 * kCus) * 64) return {kInt8Tiles256, 1};
    return {kInt8Tiles128, 1};
}

inline size_t int8_part_bytes(int rows, int n, int k, bool gated) {
    const Int8Plan p = int8_plan(rows, n, k, gated);
    return p.splits > 1 ? (size_t)p.splits * rows * int8_part_cols(n, gated) * sizeof(int) : 0;
}

// Whether the kernel of few rows quantizes `rows` rows of k columns itself.
bool int8_few_quantizes(int rows, int k);
void launch_int8_few(const Int8Args& a, hipStream_t stream);
void launch_int8_tiles(const Int8Args& a, const Int8Plan& plan, hipStream_t stream);

}  // namespace dmoe
