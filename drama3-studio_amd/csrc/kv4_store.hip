// Rows into the 4-bit paged cache (rotation by position and quantization on
// the way) and back out of it.
//
// Mathematics of the quantizer, for the 32 values x of a scale word: with
// r = max(x, 0) - min(x, 0), the scale s is the smallest number of seven
// significant bits with 15 s >= r, the zero point z = rint(-min(x, 0) / s) and
// a code rint(x / s) + z, cut to 0..15.  Quotients are rounded half to even
// exactly (a remainder formed by one fma decides next to a border), so the
// codes depend on x alone and not on how a division is carried out.  Keys are
// rotated in 64 bits and rounded once to 32: angles of far positions keep
// their digits, and codes do not change with the order of operations.
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "kernels.hpp"
#include "kv4.hpp"

namespace dmoe {
namespace {

constexpr int kThreads = 256;
// Rows go eight to a workgroup where one by one they would make eight times
// this many workgroups of 256 threads: with fewer the chip is not full (2300
// rows of 20 heads of 256 channels: 6900 workgroups, 21 us one by one, 25 us by
// eight; 8192 rows of 48 heads of 128: 24576, 74 us one by one, 55 by eight).
constexpr int kFull = 1024;

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Where a row's token is kept.
struct Place {
    uint8_t* page;  // null: a table entry names no page
    int pos;        // place in the sequence, -1 if no sequence owns the row or it has none
};

// Every lane of the wave calls this with the same row.
__device__ __forceinline__ Place place_of(const Kv4Cache& c, const Kv4Batch& b, int row, int* status) {
    Place none{nullptr, -1};
    if (row >= b.rows) return none;
    int seq = row;
    if (b.starts) {
        seq = 0;
        const int lane = threadIdx.x & 63;
        for (int s = 0; s < b.seqs; s += kWave)
            seq += __popcll(__ballot(s + lane < b.seqs && b.starts[min(s + lane, b.seqs - 1) + 1] <= row));
    }
    if (seq >= b.seqs) return none;
    bool bad;
    const Kv4Seq q = kv4_seq(b, c.page_shift, seq, bad);
    if (bad && status && !b.starts) raise_status(status, kBadBatch);
    const int pos = q.len - q.n + (row - q.row0);
    if (row < q.row0 || row >= q.row0 + q.n || pos < 0) return none;
    const int page = b.table[(int64_t)seq * b.table_stride + (pos >> c.page_shift)];
    const bool off = (unsigned)page >= (unsigned)c.num_pages;
    if (off && status) raise_status(status, kBadBatch);
    return Place{off ? nullptr : c.pages + (int64_t)page * c.page_stride, pos};
}

// Reports a batch's bad sequences, also those that none of the buffers' rows
// belongs to: the last wave of one workgroup, beside the wave that finds a
// row's place.
__device__ __forceinline__ void report_sequences(const Kv4Cache& c, const Kv4Batch& b, int* status) {
    if (!b.starts || !status || blockIdx.x || blockIdx.y || wave_index() != (int)blockDim.x / kWave - 1) return;
    for (int s = threadIdx.x & 63; s < b.seqs; s += kWave) {
        bool bad;
        kv4_seq(b, c.page_shift, s, bad);
        if (bad) raise_status(status, kBadBatch);
    }
}

typedef _Float16 v8h __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void unpack8(const v4i& raw, int dtype, float (&x)[8]) {
    if (dtype == kBF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float((uint32_t)raw[i] << 16);
            x[2 * i + 1] = __uint_as_float((uint32_t)raw[i] & 0xFFFF0000u);
        }
    } else {
        const v8h h = __builtin_bit_cast(v8h, raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
    }
}

__device__ __forceinline__ v4i pack8(const float (&x)[8], int dtype) {
    if (dtype == kBF16) {
        v8bf h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = (__bf16)x[i];
        return __builtin_bit_cast(v4i, h);
    }
    v8h h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
    return __builtin_bit_cast(v4i, h);
}

// Eight codes of this lane's channels, low nibble first, and the scale word of
// the 32 channels that it shares with the three lanes beside it.
__device__ __forceinline__ uint32_t quantize8(float (&x)[8], uint32_t& scale_word, bool& odd) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);  // a NaN is the largest
    odd = most > __float_as_uint(kKv4Limit);
    if (odd) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] == x[i] ? fminf(fmaxf(x[i], -kKv4Limit), kKv4Limit) : 0.0f;
    }
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
    lo = fminf(lo, dpp_f32<kDppXor1>(lo));
    hi = fmaxf(hi, dpp_f32<kDppXor1>(hi));
    lo = fminf(lo, dpp_f32<kDppXor2>(lo));
    hi = fmaxf(hi, dpp_f32<kDppXor2>(hi));
    const float r = hi - lo;
    // the next number of the scales' grid at or above about r / 15 -- seven
    // significant bits, or fp16 subnormals without their four lowest -- and,
    // as 15 s is exact, the smallest that reaches r
    const float step = r * 0.06666667f;
    float s, less, more;
    if (step >= 0x1p-14f) {
        const uint32_t b = (__float_as_uint(step) + 0x1FFFFu) & ~0x1FFFFu;
        s = __uint_as_float(b);
        less = __uint_as_float(b - 0x20000u);
        more = __uint_as_float(b + 0x20000u);
    } else {
        s = ceilf(step * 0x1p20f) * 0x1p-20f;
        less = s - 0x1p-20f;
        more = s + 0x1p-20f;
    }
    s = 15.0f * s < r ? more : less > 0.0f && 15.0f * less >= r ? less : s;
    scale_word = 0;
    uint32_t word = 0;
    if (s > 0.0f) {
        const float y = __builtin_amdgcn_rcpf(s), middle = 0.5f * s;
        const auto quotient = [&](float v) {
            const float t = __builtin_rintf(v * y);
            const float left = __builtin_fmaf(-t, s, v), off = fabsf(left);
            const bool odd_tie = off == middle && ((int)t & 1);
            return (int)t + (off > middle || odd_tie ? (left > 0.0f ? 1 : -1) : 0);
        };
        const int z = min(quotient(-lo), 15);
        scale_word = f32_to_f16(s) | (uint32_t)z;
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= (uint32_t)max(0, min(15, quotient(x[i]) + z)) << (4 * i);
    }
    return word;
}

// Rotates the channels c0..c0+7 of a head, x; y are those half a rotation
// away, negative for the first of each pair (not used where pairs are
// neighbours).
template <class F>
__device__ __forceinline__ void rotate8(const F (&turn)[144][2], bool interleaved, int half, int c0, float (&x)[8], const float (&y)[8]) {
    if (interleaved) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const int f = (c0 + j) / 2;
            const F c = turn[f + f / 8][0], s = turn[f + f / 8][1], u = x[j], w = x[j + 1];
            x[j] = (float)(u * c - w * s);
            x[j + 1] = (float)(w * c + u * s);
        }
        return;
    }
    const int f0 = c0 - (c0 >= half ? half : 0), at = f0 + f0 / 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const F c = turn[at + j][0], s = turn[at + j][1];
        x[j] = (float)((F)x[j] * c + (F)y[j] * s);
    }
}

// kRows rows a workgroup (blockIdx.x), one 8-channel chunk of one head a
// thread: query heads first, then key and value heads.  A row alone takes
// workgroups of 256 threads, small enough that many run at once (64 rows of
// 48 heads of 128 channels: 5 us; of up to 1024 threads 8 us); eight rows take
// all their heads together, so that their angles are formed once, not three
// times, and a row's tables are read once.  8192 such rows: 55 us, 177 MB read
// and written at 3.2 TB/s, of which a third is the vector unit's (quantizer,
// 64-bit keys, angles) and the rest loads that wait for few of them.
template <int kRows>
__global__ __launch_bounds__(kRows == 1 ? kThreads : 1024) void kv4_append_kernel(Kv4AppendArgs a) {
    // cosine and sine of each frequency, in 64 bits for keys, in 32 for queries; one entry in nine is left
    // free, so that the chunks' entries lie in different banks
    __shared__ double turn[kRows][144][2];
    __shared__ float turn_q[kRows][144][2];
    __shared__ Place places[kRows];
    const int dim = a.cache.dim, chunks = dim / 8, log2 = __builtin_ctz(chunks);
    const int row0 = blockIdx.x * kRows;
    const int unit = blockIdx.y * (int)blockDim.x + threadIdx.x;
    const int head = unit >> log2, chunk = unit & (chunks - 1);
    const int kv = a.cache.kv_heads, heads = a.q_heads + 2 * kv;
    const bool is_v = head >= a.q_heads + kv, is_q = head < a.q_heads, live = head < heads;
    const int local = is_q ? head : is_v ? head - a.q_heads - kv : head - a.q_heads;
    const Kv4Rows& src = is_q ? a.q : is_v ? a.v : a.k;
    const int half = a.rotary.inv_freq ? a.rotary.dim / 2 : 0;
    const int c0 = chunk * 8;
    const bool turns = !is_v && c0 < 2 * half;
    // the lane with the other channels of the pairs; a head's lanes lie in one wave
    const int partner = (threadIdx.x & 63) + (a.rotary.interleaved ? 0 : c0 < half ? half / 8 : -(half / 8));
    v4i raw[kRows];
    if (live) {
        const uint16_t* p = (const uint16_t*)src.p + (int64_t)local * src.head_stride + c0;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const uint16_t* x = p + (int64_t)min(row0 + i, a.batch.rows - 1) * src.row_stride;
            raw[i] = *(const v4i*)x;
        }
    }
    for (int i = wave_index(); i < kRows; i += (int)blockDim.x / kWave) {
        const Place place = place_of(a.cache, a.batch, row0 + i, a.status);
        if ((threadIdx.x & 63) == 0) places[i] = place;
    }
    report_sequences(a.cache, a.batch, a.status);
    if (!a.rotary.positions) __syncthreads();
    for (int i = threadIdx.x; i < kRows * half; i += (int)blockDim.x) {
        const int row = i / half, f = i - row * half;
        double place;
        if (a.rotary.positions) {
            const int axis = a.rotary.axis ? a.rotary.axis[f] : 0;
            const int64_t at = (int64_t)min(axis, a.rotary.axes - 1) * a.rotary.axis_stride + min(row0 + row, a.batch.rows - 1);
            place = (double)load_id(a.rotary.positions, at, a.rotary.positions_dtype);
        } else {
            place = (double)places[row].pos;
        }
        const double turns_of = place * (double)a.rotary.inv_freq[f] * 0.15915494309189533577;  // 1 / (2 pi)
        double cosine, sine;
        sincospi(2.0 * (turns_of - rint(turns_of)), &sine, &cosine);
        const int at = f + f / 8;
        turn[row][at][0] = cosine;
        turn[row][at][1] = sine;
        turn_q[row][at][0] = (float)cosine;
        turn_q[row][at][1] = (float)sine;
    }
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const Place place = places[i];
        if (place.pos < 0) continue;
        float x[8];
        unpack8(raw[i], a.dtype, x);
        if (turns) {
            float y[8];
            v4i other;
#pragma unroll
            for (int j = 0; j < 4; ++j) other[j] = __shfl(raw[i][j], partner, kWave) ^ (c0 < half ? (int)0x80008000 : 0);
            unpack8(other, a.dtype, y);
            if (is_q) rotate8<float>(turn_q[i], a.rotary.interleaved, half, c0, x, y);
            else rotate8<double>(turn[i], a.rotary.interleaved, half, c0, x, y);
        }
        if (is_q) {
            uint16_t* o = (uint16_t*)a.q_out.p + (int64_t)(row0 + i) * a.q_out.row_stride + (int64_t)local * a.q_out.head_stride;
            const v4i y = pack8(x, a.dtype);
            if (kRows > 1) __builtin_nontemporal_store(y, (v4i*)(o + c0));  // more than a cache holds: 62 us with the read back, 70 without
            else *(v4i*)(o + c0) = y;
            continue;
        }
        uint32_t scale_word;
        bool odd;
        const uint32_t word = quantize8(x, scale_word, odd);
        if (odd && a.status) raise_status(a.status, kNonFinite);
        if (!place.page) continue;
        const int size = 1 << a.cache.page_shift, slot = place.pos & (size - 1);
        uint8_t* base = place.page + local * kv4_head_bytes(size, dim);
        uint16_t* scales = (uint16_t*)(base + (int64_t)size * dim) + (is_v ? size * (dim / kKv4Group) : 0);
        if (is_v) ((uint32_t*)(base + size * dim / 2))[(slot / 4 * chunks + chunk) * 4 + slot % 4] = word;
        else ((uint32_t*)base)[slot * chunks + chunk] = word;
        if (chunk % 4 == 0) scales[chunk / 4 * size + slot] = (uint16_t)scale_word;
    }
}

// kRows rows a workgroup, one 8-channel chunk of a key or value head a thread:
// bound by memory.  Rows are written past the caches (30001 rows of 8 + 8
// heads of 128 channels, 157 MB: 31 us, 5.1 TB/s, more than a copy reaches;
// 50 us with ordinary stores).
template <int kRows>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(Kv4ReadArgs a) {
    __shared__ Place places[kRows];
    const int dim = a.cache.dim, chunks = dim / 8, log2 = __builtin_ctz(chunks), kv = a.cache.kv_heads;
    const int row0 = blockIdx.x * kRows;
    const int unit = blockIdx.y * kThreads + threadIdx.x;
    const int head = unit >> log2, chunk = unit & (chunks - 1);
    const bool is_v = head >= kv, live = head < 2 * kv;
    const int local = is_v ? head - kv : head;
    for (int i = wave_index(); i < kRows; i += kThreads / kWave) {
        const Place place = place_of(a.cache, a.batch, row0 + i, a.status);
        if ((threadIdx.x & 63) == 0) places[i] = place;
    }
    report_sequences(a.cache, a.batch, a.status);
    __syncthreads();
    if (!live) return;
    const int size = 1 << a.cache.page_shift;
    const int64_t head_at = local * kv4_head_bytes(size, dim);
    uint32_t word[kRows], scale[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        word[i] = scale[i] = 0;
        const Place place = places[i];
        if (!place.page) continue;
        const int slot = place.pos & (size - 1);
        const uint8_t* base = place.page + head_at;
        const uint16_t* scales = (const uint16_t*)(base + (int64_t)size * dim) + (is_v ? size * (dim / kKv4Group) : 0);
        word[i] = is_v ? ((const uint32_t*)(base + size * dim / 2))[(slot / 4 * chunks + chunk) * 4 + slot % 4]
                       : ((const uint32_t*)base)[slot * chunks + chunk];
        scale[i] = scales[chunk / 4 * size + slot];
    }
    const Kv4Rows& dst = is_v ? a.v : a.k;
    uint16_t* o = (uint16_t*)dst.p + (int64_t)local * dst.head_stride + chunk * 8;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (places[i].pos < 0) continue;
        const float s = f16_to_f32(scale[i] & 0xFFF0);
        const int z = scale[i] & 15;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)((int)(word[i] >> (4 * j) & 15) - z) * s;
        __builtin_nontemporal_store(pack8(x, a.dtype), (v4i*)(o + (int64_t)(row0 + i) * dst.row_stride));
    }
}

}  // namespace

void launch_kv4_append(const Kv4AppendArgs& a, hipStream_t st) {
    const int units = (a.q_heads + 2 * a.cache.kv_heads) * (a.cache.dim / 8);
    const int small = (units + kThreads - 1) / kThreads;
    if ((int64_t)a.batch.rows * small < 8 * kFull) {
        kv4_append_kernel<1><<<dim3(a.batch.rows, small), kThreads, 0, st>>>(a);
        return;
    }
    const int parts = (units + 1023) / 1024, threads = ((units + parts - 1) / parts + kWave - 1) / kWave * kWave;
    kv4_append_kernel<8><<<dim3((a.batch.rows + 7) / 8, parts), threads, 0, st>>>(a);
}

void launch_kv4_read(const Kv4ReadArgs& a, hipStream_t st) {
    const int units = 2 * a.cache.kv_heads * (a.cache.dim / 8);
    const unsigned parts = (units + kThreads - 1) / kThreads;
    if ((int64_t)a.batch.rows * parts < 8 * kFull) kv4_read_kernel<1><<<dim3(a.batch.rows, parts), kThreads, 0, st>>>(a);
    else kv4_read_kernel<8><<<dim3((a.batch.rows + 7) / 8, parts), kThreads, 0, st>>>(a);
}

}  // namespace dmoe
