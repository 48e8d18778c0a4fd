// Device helpers of rows in 8 bits: loads of eight columns at any alignment
// and the roundings to 8-bit integers and E4M3 that are right at every border.
#pragma once

#include "common.hpp"
#include "int8.hpp"

namespace dmoe {

// Rows of an odd width begin at any element: the type tells the compiler, and
// the hardware takes such 16-byte accesses.
struct __attribute__((packed, aligned(2))) Any16 {
    uint32_t w[4];
};

template <int DT>
__device__ __forceinline__ constexpr int elem_bytes() { return DT == kF32 ? 4 : 2; }

// Columns [col, col + 8) of a row as fp32, zeros from `cols` on.
template <int DT>
__device__ __forceinline__ void load_cols8(const void* row, int col, int cols, float* v) {
    if (col + 8 <= cols) {
        const char* p = (const char*)row + (int64_t)col * elem_bytes<DT>();
        if constexpr (DT == kF32) {
            const Any16 a = *(const Any16*)p, b = *(const Any16*)(p + 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = __uint_as_float(a.w[j]);
                v[4 + j] = __uint_as_float(b.w[j]);
            }
        } else {
            const Any16 a = *(const Any16*)p;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint16_t lo = (uint16_t)a.w[j], hi = (uint16_t)(a.w[j] >> 16);
                v[2 * j] = DT == kBF16 ? bf16_to_f32(lo) : f16_to_f32(lo);
                v[2 * j + 1] = DT == kBF16 ? bf16_to_f32(hi) : f16_to_f32(hi);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = col + j < cols ? load_as_f32(row, col + j, DT) : 0.0f;
    }
}

// Two values rounded to a 16-bit type by the hardware's conversion (for bf16 one instruction for both).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (DT == kBF16) {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2{(__bf16)lo, (__bf16)hi});
    } else {
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2{(_Float16)lo, (_Float16)hi});
    }
}

// Eight values to where they lie; past the caches, whose lines the call itself has no more use for.
template <int DT>
__device__ __forceinline__ void put_cols8(void* p, const float* v) {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    typedef v4u any16 __attribute__((aligned(2)));
    if constexpr (DT == kF32) {
        __builtin_nontemporal_store(v4u{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])},
                                    (any16*)p);
        __builtin_nontemporal_store(v4u{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])},
                                    (any16*)p + 1);
    } else {
        __builtin_nontemporal_store(v4u{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])},
                                    (any16*)p);
    }
}

template <int DT>
__device__ __forceinline__ void store_cols8(void* row, int col, int cols, const float* v) {
    if (col + 8 <= cols) {
        put_cols8<DT>((char*)row + (int64_t)col * elem_bytes<DT>(), v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + j < cols) store_from_f32(row, col + j, DT, v[j]);
    }
}

// |v| as bits: ordered as the values, an infinity above every number and a NaN
// above that, so that an integer maximum loses neither.
__device__ __forceinline__ int magnitude(float v) { return __float_as_int(v) & 0x7FFFFFFF; }

__device__ __forceinline__ int row_max_bits(int v) {
    v = max(v, dpp_i32<kDppXor1>(v));
    v = max(v, dpp_i32<kDppXor2>(v));
    v = max(v, dpp_i32<kDppHalfMirror>(v));
    return max(v, dpp_i32<kDppMirror>(v));
}
__device__ __forceinline__ int wave_max_bits(int v) {
    v = row_max_bits(v);
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

__device__ __forceinline__ bool finite_bits(float v) { return magnitude(v) < 0x7F800000; }

// Eight values u * by in units of `scale`, rounded to the nearest integers.
// The 32-bit quotient is off by less than 2^-15 (a product of at most 127
// with two roundings of 2^-24), so only one closer than 2^-14 to the middle
// between two integers needs the 64-bit one; `each` is by / scale in 32 bits.
__device__ __forceinline__ uint64_t int8_codes8(const float* u, float each, double by, float scale) {
    float t[8], close = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float f = u[j] * each;
        t[j] = __builtin_rintf(f);
        close = fmaxf(close, fabsf(f - t[j]));
    }
    if (close > 0.5f - 0x1p-14f) {
#pragma unroll 1
        for (int j = 0; j < 8; ++j) t[j] = (float)__builtin_rint((double)u[j] * by / (double)scale);
    }
    uint64_t q = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int c = (int)fminf(fmaxf(t[j], -127.0f), 127.0f);
        q |= (uint64_t)(uint8_t)c << (8 * j);
    }
    return q;
}

// Eight values u * by in units of `scale` as the nearest E4M3 numbers, beyond
// +-448 that.  Every number and every middle of two is a multiple of 2^19 in
// the bits of an fp32 value; a quotient within four steps of one is formed in
// 64 bits and kept off the middle that it is not (its last bit set).
__device__ __forceinline__ uint64_t e4m3_codes8(const float* u, float each, double by, float scale) {
    float f[8];
    bool close = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        f[j] = u[j] * each;
        close |= ((__float_as_uint(f[j]) + 4u) & 0x7FFFFu) <= 8u;
    }
    if (close) {
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
            const double d = (double)u[j] * by / (double)scale;
            uint32_t bits = __float_as_uint((float)d);
            const double back = (double)__uint_as_float(bits);
            // rounded away from zero past d: the number below it; then odd, which no middle is
            if (fabs(back) > fabs(d)) bits -= 1;
            if (back != d) bits |= 1;
            f[j] = __uint_as_float(bits);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = fminf(fmaxf(f[j], -448.0f), 448.0f);
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], hi, true);
    return (uint32_t)lo | (uint64_t)(uint32_t)hi << 32;
}

// Scale of rows (groups) whose largest magnitude is `top`.
__device__ __forceinline__ float int8_scale(float top) { return fmaxf(top, 1e-12f) * (1.0f / 127.0f); }
__device__ __forceinline__ float e4m3_scale(float top) { return fmaxf(top, 1e-10f) * (1.0f / 448.0f); }

}  // namespace dmoe
