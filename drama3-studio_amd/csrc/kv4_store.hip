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

// The sequence that owns row `row`, and the row's place in its cache; false if
// no sequence owns it.  Every lane of the wave calls this with the same row.
__device__ __forceinline__ bool locate_row(const Kv4Batch& b, int page_shift, int row, int* status, int& seq, int& pos) {
    seq = row;
    if (b.starts) {
        seq = 0;
        for (int s = threadIdx.x & 63; s - (int)(threadIdx.x & 63) < b.seqs; s += kWave)
            seq += __popcll(__ballot(s < b.seqs && b.starts[min(s, b.seqs - 1) + 1] <= row));
    }
    if (seq >= b.seqs) return false;
    bool bad;
    const Kv4Seq q = kv4_seq(b, page_shift, seq, bad);
    if (bad && status) raise_status(status, kBadBatch);
    pos = q.len - q.n + (row - q.row0);
    return row >= q.row0 && row < q.row0 + q.n && pos >= 0;
}

// Page and slot of a token, or null where its table entry names no page.
__device__ __forceinline__ uint8_t* token_page(const Kv4Cache& c, const Kv4Batch& b, int seq, int pos, int* status) {
    const int page = b.table[(int64_t)seq * b.table_stride + (pos >> c.page_shift)];
    if ((unsigned)page >= (unsigned)c.num_pages) {
        if (status) raise_status(status, kBadBatch);
        return nullptr;
    }
    return c.pages + (int64_t)page * c.page_stride;
}

__device__ __forceinline__ void unpack8(const v4i& raw, int dtype, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = (uint32_t)raw[i];
        x[2 * i] = dtype == kBF16 ? bf16_to_f32(w & 0xFFFF) : f16_to_f32(w & 0xFFFF);
        x[2 * i + 1] = dtype == kBF16 ? bf16_to_f32(w >> 16) : f16_to_f32(w >> 16);
    }
}

__device__ __forceinline__ v4i pack8(const float (&x)[8], int dtype) {
    v4i raw;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        raw[i] = dtype == kBF16 ? (int)(f32_to_bf16(x[2 * i]) | (uint32_t)f32_to_bf16(x[2 * i + 1]) << 16)
                                : (int)(f32_to_f16(x[2 * i]) | (uint32_t)f32_to_f16(x[2 * i + 1]) << 16);
    return raw;
}

// Eight codes of this lane's channels, low nibble first, and the scale word of
// the 32 channels that it shares with the three lanes beside it.
__device__ __forceinline__ uint32_t quantize8(float (&x)[8], uint32_t& scale_word, bool& odd) {
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = x[i] == x[i] ? fminf(fmaxf(x[i], -kKv4Limit), kKv4Limit) : 0.0f;
        odd |= v != x[i];
        x[i] = v;
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    lo = fminf(lo, dpp_f32<kDppXor1>(lo));
    hi = fmaxf(hi, dpp_f32<kDppXor1>(hi));
    lo = fminf(lo, dpp_f32<kDppXor2>(lo));
    hi = fmaxf(hi, dpp_f32<kDppXor2>(hi));
    const float r = hi - lo;
    const float step = r / 15.0f;
    float s;
    if (step >= 0x1p-14f) {  // up to seven significant bits
        s = __uint_as_float((__float_as_uint(step) + 0x1FFFFu) & ~0x1FFFFu);
        if (15.0f * s < r) s = __uint_as_float(__float_as_uint(s) + 0x20000u);
    } else {  // fp16 subnormals without their four lowest bits
        s = ceilf(step * 0x1p20f) * 0x1p-20f;
        if (15.0f * s < r) s += 0x1p-20f;
    }
    scale_word = 0;
    uint32_t word = 0;
    if (s > 0.0f) {
        const float y = 1.0f / s;
        const auto quotient = [&](float v) {
            float t = __builtin_rintf(v * y);
            const float left = __builtin_fmaf(-t, s, v), two = 2.0f * fabsf(left);
            if (two > s || (two == s && ((int)t & 1))) t += left > 0.0f ? 1.0f : -1.0f;
            return (int)t;
        };
        const int z = min(quotient(-lo), 15);
        scale_word = f32_to_f16(s) | (uint32_t)z;
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= (uint32_t)max(0, min(15, quotient(x[i]) + z)) << (4 * i);
    }
    return word;
}

// One row a workgroup (blockIdx.x), one 8-channel chunk of one head a thread:
// query heads first, then key and value heads.
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(Kv4AppendArgs a) {
    __shared__ double turn[128][2];
    const int dim = a.cache.dim, chunks = dim / 8;
    const int row = blockIdx.x;
    int seq, pos;
    if (!locate_row(a.batch, a.cache.page_shift, row, a.status, seq, pos)) return;
    const int unit = blockIdx.y * kThreads + threadIdx.x;
    const int head = unit / chunks, chunk = unit % chunks;
    const int kv = a.cache.kv_heads, heads = a.q_heads + 2 * kv;
    const bool is_v = head >= a.q_heads + kv, is_q = head < a.q_heads, live = head < heads;
    const int local = is_q ? head : is_v ? head - a.q_heads - kv : head - a.q_heads;
    const Kv4Rows& src = is_q ? a.q : is_v ? a.v : a.k;
    const int half = a.rotary.inv_freq ? a.rotary.dim / 2 : 0;
    const int c0 = chunk * 8;
    const bool turns = !is_v && c0 < 2 * half;
    const bool apart = turns && !a.rotary.interleaved;  // the other channels of the pairs lie half a rotation away
    v4i raw = {0, 0, 0, 0}, other = {0, 0, 0, 0};
    if (live) {
        const uint16_t* p = (const uint16_t*)src.p + (int64_t)row * src.row_stride + (int64_t)local * src.head_stride;
        raw = *(const v4i*)(p + c0);
        if (apart) other = *(const v4i*)(p + (c0 < half ? c0 + half : c0 - half));
    }
    for (int i = threadIdx.x; i < half; i += kThreads) {
        double place = pos;
        if (a.rotary.positions) {
            const int axis = a.rotary.axis ? a.rotary.axis[i] : 0;
            const int64_t at = (int64_t)min(axis, a.rotary.axes - 1) * a.rotary.axis_stride + row;
            place = (double)load_id(a.rotary.positions, at, a.rotary.positions_dtype);
        }
        const double turns_of = place * (double)a.rotary.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
        sincospi(2.0 * (turns_of - rint(turns_of)), &turn[i][1], &turn[i][0]);
    }
    __syncthreads();
    if (!live) return;
    float x[8];
    unpack8(raw, a.dtype, x);
    if (turns) {
        float y[8];
        unpack8(other, a.dtype, y);
        const bool second = c0 >= half;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if (apart) {
                const double* t0 = turn[c0 + i - (second ? half : 0)];
                const double* t1 = turn[c0 + i + 1 - (second ? half : 0)];
                const double s0 = second ? t0[1] : -t0[1], s1 = second ? t1[1] : -t1[1];
                x[i] = (float)((double)x[i] * t0[0] + (double)y[i] * s0);
                x[i + 1] = (float)((double)x[i + 1] * t1[0] + (double)y[i + 1] * s1);
            } else {
                const double* t = turn[(c0 + i) / 2];
                const double u = x[i], w = x[i + 1];
                x[i] = (float)(u * t[0] - w * t[1]);
                x[i + 1] = (float)(w * t[0] + u * t[1]);
            }
        }
    }
    if (is_q) {
        uint16_t* o = (uint16_t*)a.q_out.p + (int64_t)row * a.q_out.row_stride + (int64_t)local * a.q_out.head_stride;
        *(v4i*)(o + c0) = pack8(x, a.dtype);
        return;
    }
    uint8_t* page = token_page(a.cache, a.batch, seq, pos, a.status);
    uint32_t scale_word;
    bool odd = false;
    const uint32_t word = quantize8(x, scale_word, odd);
    if (odd && a.status) raise_status(a.status, kNonFinite);
    if (!page) return;
    const int size = 1 << a.cache.page_shift, slot = pos & (size - 1);
    uint8_t* base = page + local * kv4_head_bytes(size, dim);
    uint16_t* scales = (uint16_t*)(base + (int64_t)size * dim) + (is_v ? size * (dim / kKv4Group) : 0);
    if (is_v) ((uint32_t*)(base + size * dim / 2))[(slot / 4 * chunks + chunk) * 4 + slot % 4] = word;
    else ((uint32_t*)base)[slot * chunks + chunk] = word;
    if (chunk % 4 == 0) scales[chunk / 4 * size + slot] = (uint16_t)scale_word;
}

// One row a workgroup, one 8-channel chunk of a key or value head a thread.
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(Kv4ReadArgs a) {
    const int dim = a.cache.dim, chunks = dim / 8, kv = a.cache.kv_heads;
    const int row = blockIdx.x;
    int seq, pos;
    if (!locate_row(a.batch, a.cache.page_shift, row, a.status, seq, pos)) return;
    const int unit = blockIdx.y * kThreads + threadIdx.x;
    const int head = unit / chunks, chunk = unit % chunks;
    if (head >= 2 * kv) return;
    const bool is_v = head >= kv;
    const int local = is_v ? head - kv : head;
    const uint8_t* page = token_page(a.cache, a.batch, seq, pos, a.status);
    float x[8] = {};
    if (page) {
        const int size = 1 << a.cache.page_shift, slot = pos & (size - 1);
        const uint8_t* base = page + local * kv4_head_bytes(size, dim);
        const uint16_t* scales = (const uint16_t*)(base + (int64_t)size * dim) + (is_v ? size * (dim / kKv4Group) : 0);
        const uint32_t word = is_v ? ((const uint32_t*)(base + size * dim / 2))[(slot / 4 * chunks + chunk) * 4 + slot % 4]
                                   : ((const uint32_t*)base)[slot * chunks + chunk];
        const uint32_t sw = scales[chunk / 4 * size + slot];
        const float s = f16_to_f32(sw & 0xFFF0);
        const int z = sw & 15;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)((int)(word >> (4 * i) & 15) - z) * s;
    }
    const Kv4Rows& dst = is_v ? a.v : a.k;
    uint16_t* o = (uint16_t*)dst.p + (int64_t)row * dst.row_stride + (int64_t)local * dst.head_stride;
    *(v4i*)(o + chunk * 8) = pack8(x, a.dtype);
}

}  // namespace

void launch_kv4_append(const Kv4AppendArgs& a, hipStream_t st) {
    const int units = (a.q_heads + 2 * a.cache.kv_heads) * (a.cache.dim / 8);
    const dim3 grid(a.batch.rows, (units + kThreads - 1) / kThreads);
    kv4_append_kernel<<<grid, kThreads, 0, st>>>(a);
}

void launch_kv4_read(const Kv4ReadArgs& a, hipStream_t st) {
    const int units = 2 * a.cache.kv_heads * (a.cache.dim / 8);
    const dim3 grid(a.batch.rows, (units + kThreads - 1) / kThreads);
    kv4_read_kernel<<<grid, kThreads, 0, st>>>(a);
}

}  // namespace dmoe
