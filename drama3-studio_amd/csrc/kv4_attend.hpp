// Device helpers of the attention kernels over the 4-bit cache.
//
// Codes become fp16 without conversions: a nibble put into the mantissa of
// 1024 (low) or 64 (high) is 1024 + c or 64 + c, from which 1024 + z or 64 + z
// is taken exactly; times s it is exact again.  Queries are scaled by a power
// of two per row into fp16, the row's largest channel to [0.5, 1): channels of
// 2^-14 of that power (fp16 rows; 2^-17 for bf16, which has fewer digits) keep
// all their digits, smaller ones become multiples of 2^-24 of it.  So a score
// is at most 2^-25 of the power times the sum of its |k| off, times the scale.
// P is shifted by 2^8, which keeps weights down to 2^-22 normal, and is rounded
// to fp16 with the sums in fp32.
#pragma once

#include "common.hpp"
#include "kv4_plan.hpp"

namespace dmoe {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr float kKv4Shift = 8.0f;  // P is held times 2^8; 2^16 is where fp16 ends

__device__ __forceinline__ v2h as_h2(uint32_t w) { return __builtin_bit_cast(v2h, w); }

// The two masks and biases of a code pair's bits, held in registers: an
// instruction takes only one constant of its own.
struct CodeBits {
    uint32_t low_mask, high_mask, low_bias, high_bias;
};
__device__ __forceinline__ CodeBits code_bits() {
    CodeBits k{0x000F000Fu, 0x00F000F0u, 0x64006400u, 0x54005400u};
    asm("" : "+s"(k.low_mask), "+s"(k.high_mask), "+v"(k.low_bias), "+v"(k.high_bias));
    return k;
}

// fp16 pairs of the low (+0) and high (+1) nibbles of w's two low bytes of
// each half, less the zero points, times the scales.
__device__ __forceinline__ v2h low_pair(const CodeBits& k, uint32_t w, v2h zero, v2h scale) {
    return (as_h2((w & k.low_mask) | k.low_bias) - zero) * scale;
}
__device__ __forceinline__ v2h high_pair(const CodeBits& k, uint32_t w, v2h zero, v2h scale) {
    return (as_h2((w & k.high_mask) | k.high_bias) - zero) * scale;
}

// The scale words of two tokens (or one, in both halves) as operands of the above.
struct Scales {
    v2h scale, low_zero, high_zero;
};
__device__ __forceinline__ Scales scales_of(const CodeBits& k, uint32_t words) {
    const uint32_t z = words & k.low_mask;
    return Scales{as_h2(words ^ z), as_h2(z | k.low_bias), as_h2(z << 4 | k.high_bias)};
}

__device__ __forceinline__ v8h join(v2h a, v2h b, v2h c, v2h d) {
    return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Two values as a word of a bf16 or fp16 row.
__device__ __forceinline__ uint32_t narrow2(float a, float b, int dtype) {
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    return dtype == kBF16 ? __builtin_bit_cast(uint32_t, v2bf{(__bf16)a, (__bf16)b})
                          : __builtin_bit_cast(uint32_t, v2h{(_Float16)a, (_Float16)b});
}

// A query row of which this lane holds N words of eight channels: to fp16
// by the power of two that brings the row's largest value `most` to [0.5, 1),
// channels in the order in which low_pair / high_pair take a code word's.
// Returns the factor that takes the scores back, times scale_log2.
template <int N>
__device__ __forceinline__ float scale_query(const v4i (&raw)[N], float most, int dtype, float scale_log2, v8h (&query)[N]) {
    int e = 0;
    if (most > 0.0f && most < __builtin_inff()) (void)frexpf(most, &e);
    e = max(-120, min(120, e));
    // an infinity or NaN makes all of the row's scores no number: else an infinity whose
    // scores are all minus infinity would look like a row that sees nothing
    const float down = most < __builtin_inff() ? ldexpf(1.0f, -e) : __builtin_nanf("");
    const auto fill = [&](auto&& element) {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // channels i and i + 4
                query[j][2 * i] = (_Float16)(element(j, i) * down);
                query[j][2 * i + 1] = (_Float16)(element(j, i + 4) * down);
            }
    };
    if (dtype == kBF16) {
        fill([&](int j, int i) { return __uint_as_float(i & 1 ? (uint32_t)raw[j][i / 2] & 0xFFFF0000u : (uint32_t)raw[j][i / 2] << 16); });
    } else {
        fill([&](int j, int i) { return (float)as_h2((uint32_t)raw[j][i / 2])[i & 1]; });
    }
    return fmaxf(scale_log2 * ldexpf(1.0f, e), 1e-35f);
}

// The largest magnitude of a query row's words, found among their bits: those
// of both types grow with it (NaN above all).
template <int N>
__device__ __forceinline__ float largest(const v4i (&raw)[N], int dtype) {
    typedef uint16_t v2s __attribute__((ext_vector_type(2)));
    v2s most{0, 0};
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            most = __builtin_elementwise_max(most, __builtin_bit_cast(v2s, (uint32_t)raw[j][i] & 0x7FFF7FFFu));
    const uint32_t top = max((uint32_t)most[0], (uint32_t)most[1]);
    return dtype == kBF16 ? __uint_as_float(top << 16) : (float)as_h2(top)[0];
}

// Largest / sum over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float groups_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

}  // namespace dmoe
