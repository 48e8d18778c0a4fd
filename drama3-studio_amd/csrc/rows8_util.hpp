// Device helpers of rows in 8 bits: loads of eight columns at any alignment
// and the roundings to 8-bit integers and E4M3 that are right at every border.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "int8.hpp"

namespace dmoe {

// Rows of an odd width begin at any element: the type tells the compiler, and
// the hardware takes such 16-byte accesses.
struct __attribute__((packed, aligned(2))) Any16 {
    uint32_t w[4];
};

template <int DT>
__host__ __device__ __forceinline__ constexpr int elem_bytes() { return DT == kF32 ? 4 : 2; }

// Eight columns of a row in its type.
template <int DT>
struct Cols8 {
    uint32_t w[DT == kF32 ? 8 : 4];
};

template <int DT>
__device__ __forceinline__ float col_of(const Cols8<DT>& c, int j) {
    if constexpr (DT == kF32) return __uint_as_float(c.w[j]);
    else if constexpr (DT == kBF16) return __uint_as_float(j % 2 ? c.w[j / 2] & 0xFFFF0000u : c.w[j / 2] << 16);
    else return f16_to_f32((uint16_t)(c.w[j / 2] >> (j % 2 * 16)));
}

// Columns [col, col + 8) of a row, zeros from `cols` on.  A row's last columns
// come with those before them, in one load, and are moved down.
template <int DT>
__device__ __forceinline__ Cols8<DT> load_raw8(const void* row, int col, int cols) {
    Cols8<DT> c = {};
    if (col >= cols) return c;
    if (cols < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < cols) {
                if constexpr (DT == kF32) c.w[j] = ((const uint32_t*)row)[j];
                else c.w[j / 2] |= (uint32_t)((const uint16_t*)row)[j] << (j % 2 * 16);
            }
        return c;
    }
    const int down = max(col + 8 - cols, 0);  // 0 to 7
    const char* p = (const char*)row + (int64_t)(col - down) * elem_bytes<DT>();
    if constexpr (DT == kF32) {
        const Any16 a = *(const Any16*)p, b = *(const Any16*)(p + 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            c.w[j] = a.w[j];
            c.w[4 + j] = b.w[j];
        }
        if (down) {
#pragma unroll
            for (int bit = 1; bit < 8; bit <<= 1)
#pragma unroll
                for (int j = 0; j < 8; ++j) c.w[j] = down & bit ? (j + bit < 8 ? c.w[j + bit] : 0u) : c.w[j];
        }
    } else {
        const Any16 a = *(const Any16*)p;
#pragma unroll
        for (int j = 0; j < 4; ++j) c.w[j] = a.w[j];
        if (down) {
#pragma unroll
            for (int words = 2; words > 0; words >>= 1)
#pragma unroll
                for (int j = 0; j < 4; ++j) c.w[j] = (down >> 1) & words ? (j + words < 4 ? c.w[j + words] : 0u) : c.w[j];
            if (down & 1) {
#pragma unroll
                for (int j = 0; j < 4; ++j) c.w[j] = c.w[j] >> 16 | (j < 3 ? c.w[j + 1] << 16 : 0u);
            }
        }
    }
    return c;
}

template <int DT>
__device__ __forceinline__ void load_cols8(const void* row, int col, int cols, float* v) {
    const Cols8<DT> c = load_raw8<DT>(row, col, cols);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col_of<DT>(c, j);
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

// Eight values in the row's type.
template <int DT>
__device__ __forceinline__ Cols8<DT> cols_of(const float* v) {
    Cols8<DT> c;
    if constexpr (DT == kF32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c.w[j] = __float_as_uint(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) c.w[j] = pack2<DT>(v[2 * j], v[2 * j + 1]);
    }
    return c;
}

// Eight columns to where they lie, past the caches, so that they do not push out what other rows are read from (us, with
// plain stores in brackets): the norm of 2000 x 4096 rows 11.8 (14.8), a product of 4096 cubed 57.0 (58.7).  What the next
// launch reads gains nothing from plain stores either: one to 509 rows the same within 1%, norm, product and norm behind
// one another 10.7 (10.7) at 13 x 2048 and 110.1 (108.9) at 4096 x 4096; hidden rows, which the feed-forward block's second
// product quantizes, 47 x 11008 38.3 for the block (38.4) and 4096 x 12288 537 (540).
template <int DT>
__device__ __forceinline__ void put_raw8(void* p, const Cols8<DT>& c) {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    typedef v4u any16 __attribute__((aligned(2)));
#pragma unroll
    for (int h = 0; h < (DT == kF32 ? 2 : 1); ++h)
        __builtin_nontemporal_store(v4u{c.w[4 * h], c.w[4 * h + 1], c.w[4 * h + 2], c.w[4 * h + 3]}, (any16*)p + h);
}
template <int DT>
__device__ __forceinline__ void put_cols8(void* p, const float* v) { put_raw8<DT>(p, cols_of<DT>(v)); }

template <int DT>
__device__ __forceinline__ void store_raw8(void* row, int col, int cols, const Cols8<DT>& c) {
    if (col + 8 <= cols) {
        put_raw8<DT>((char*)row + (int64_t)col * elem_bytes<DT>(), c);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + j < cols) {
                if constexpr (DT == kF32) ((uint32_t*)row)[col + j] = c.w[j];
                else ((uint16_t*)row)[col + j] = (uint16_t)(c.w[j / 2] >> (j % 2 * 16));
            }
    }
}
template <int DT>
__device__ __forceinline__ void store_cols8(void* row, int col, int cols, const float* v) {
    store_raw8<DT>(row, col, cols, cols_of<DT>(v));
}

// |v| as bits: ordered as the values, an infinity above every number and a NaN
// above that, so that an integer maximum loses neither.
__device__ __forceinline__ int magnitude(float v) { return __float_as_int(v) & 0x7FFFFFFF; }

// The largest of eight columns, as magnitude() has it: of 16-bit types two at a time.
template <int DT>
__device__ __forceinline__ int magnitude8(const Cols8<DT>& c) {
    int m = 0;
    if constexpr (DT == kF32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, (int)(c.w[j] & 0x7FFFFFFFu));
    } else {
        typedef uint16_t v2 __attribute__((ext_vector_type(2)));
        v2 top = {0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(v2, c.w[j] & 0x7FFF7FFFu));
        const uint16_t t = max(top[0], top[1]);
        m = DT == kBF16 ? (int)t << 16 : magnitude(f16_to_f32(t));
    }
    return m;
}

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

__device__ __forceinline__ double row_sum_f64(double v) {
    const auto add = [&](auto ctrl) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)dpp_i32<decltype(ctrl)::value>((int)(uint32_t)b);
        const uint32_t hi = (uint32_t)dpp_i32<decltype(ctrl)::value>((int)(uint32_t)(b >> 32));
        v += __builtin_bit_cast(double, lo | (uint64_t)hi << 32);
    };
    add(std::integral_constant<int, kDppXor1>{});
    add(std::integral_constant<int, kDppXor2>{});
    add(std::integral_constant<int, kDppHalfMirror>{});
    add(std::integral_constant<int, kDppMirror>{});
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v = row_sum_f64(v);
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    double s = 0.0;
#pragma unroll
    for (int l = 0; l < kWave; l += 16) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
        s += __builtin_bit_cast(double, lo | (uint64_t)hi << 32);
    }
    return s;
}

// 1 / sqrt(x) and 1 / x to within 2^-50: the hardware's start (over 20 bits)
// and two steps of Newton's, which double them; 0, infinities and NaN give
// what the start gives.
__device__ __forceinline__ double rsqrt_f64(double x) {
    const double y0 = __builtin_amdgcn_rsq(x);
    double y = y0;
#pragma unroll
    for (int i = 0; i < 2; ++i) y = __builtin_fma(0.5 * y, __builtin_fma(-x * y, y, 1.0), y);
    return x > 0.0 && x < __builtin_inf() ? y : y0;
}
__device__ __forceinline__ double rcp_f64(double x) {
    double y = __builtin_amdgcn_rcp(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) y = __builtin_fma(y, __builtin_fma(-x, y, 1.0), y);
    return y;
}

// What codes are formed from: values u stand for u * by, in units of `scale`;
// `each` is by / scale to within 2^-49.
struct Units {
    double by, each;
    float scale;
};
__device__ __forceinline__ Units units_of(double by, float scale) { return {by, by * rcp_f64((double)scale), scale}; }

// Eight values rounded to the nearest integers of their units, all within
// +-127 as the scale is the largest one's.  Added to 1.5 * 2^23, a product is
// rounded to an integer, whose low byte is the code.  The 32-bit quotient is
// off by at most 127 * 2^-24 (by.each's rounding), so only one closer than
// 2^-16 to the middle between two integers needs the 64-bit one, and only one
// of those within 2^-40 a division.
__device__ __forceinline__ uint64_t int8_codes8(const float* u, const Units& by) {
    constexpr float kMagic = 12582912.0f;
    const float each = (float)by.each;
    float t[8], close = __builtin_isinf(each) ? 0.5f : 0.0f;  // beyond 32 bits where all of a row lie below 2^-120
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        t[j] = __builtin_fmaf(u[j], each, kMagic);
        close = fmaxf(close, fabsf(__builtin_fmaf(u[j], each, kMagic - t[j])));
    }
    if (close > 0.5f - 0x1p-16f) {
        double nearest = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double d = (double)u[j] * by.each, i = __builtin_rint(d);
            t[j] = kMagic + (float)i;
            nearest = fmax(nearest, fabs(d - i));
        }
        if (nearest > 0.5 - 0x1p-40) {
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = kMagic + (float)__builtin_rint((double)u[j] * by.by / (double)by.scale);
        }
    }
    const auto four = [&](const float* v) {
        const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x0C0C0400);
        const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x0C0C0400);
        return a | b << 16;
    };
    return four(t) | (uint64_t)four(t + 4) << 32;
}

// Rounded to fp32 with the last bit set where that is not exact, so that the
// result lies on no number of fewer bits and on no middle of two.
__device__ __forceinline__ float round_to_odd(double d) {
    uint32_t bits = __float_as_uint((float)d);
    const double back = (double)__uint_as_float(bits);
    if (fabs(back) > fabs(d)) bits -= 1;
    if (back != d) bits |= 1;
    return __uint_as_float(bits);
}

// Eight values as the nearest E4M3 numbers of their units, within +-448 but for
// the quotient's last bits.
// Every number and every middle of two is a multiple of 2^19 in the bits of an
// fp32 value; only a 32-bit quotient within two steps of one (its two
// roundings) needs the 64-bit one, and only one of those within 2^-40 a division.
__device__ __forceinline__ uint64_t e4m3_codes8(const float* u, const Units& by) {
    const float each = (float)by.each;
    float f[8];
    bool close = __builtin_isinf(each);  // as above
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        f[j] = u[j] * each;
        close |= ((__float_as_uint(f[j]) + 2u) & 0x7FFFFu) <= 4u;
    }
    if (close) {
        bool on = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double d = (double)u[j] * by.each;
            const float r = (float)d;
            on |= (__float_as_uint(r) & 0x7FFFFu) == 0 && fabs((double)r - d) <= 0x1p-40 * fabs(d);
            f[j] = round_to_odd(d);
        }
        if (on) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = round_to_odd((double)u[j] * by.by / (double)by.scale);
        }
    }
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
