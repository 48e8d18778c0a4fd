// What the products of 8-bit integers make of an int32 sum.
#pragma once

#include "common.hpp"

namespace dmoe {

// A sum in units of its matrix row's scale and its activation row's, in that
// order: only a scale from 2^98 up can take the first product out of fp32's
// range where the result is in it, and then the row's comes first (a product
// below 2^-126, of a scale that is itself, is exact).  The product is rounded
// before anything is added to it, in every kernel: fused with an addition in
// one and not in another, a row's bits would depend on the size of its call.
// CHECKED false: for channels whose scale is known to be below kInt8Large.
constexpr float kInt8Large = 0x1p97f;
template <bool CHECKED = true>
__device__ __forceinline__ float int8_value(int sum, float channel, float row) {
#pragma clang fp contract(off)
    const float first = (float)sum * channel;
    if (CHECKED && __builtin_expect(__builtin_isinf(first), 0)) return (float)sum * row * channel;
    return first * row;
}

// act(z): z / (1 + exp(-z)), or gelu in its tanh form, which is
// z / (1 + exp(-2 sqrt(2 / pi) (z + 0.044715 z^3))).  The hardware's 2^x and
// reciprocal, each within 2^-23; the argument's rounding costs |y| 2^-23 more.
__device__ __forceinline__ float int8_gate(float z, int gelu) {
    constexpr float kLog2e = 1.4426950408889634f, kGelu = 1.5957691216057308f * kLog2e;
    const float y = gelu ? kGelu * __builtin_fmaf(0.044715f * z * z, z, z) : kLog2e * z;
    // 2^-y above 2^126, or an infinity, has no normal reciprocal, and the result is 0: less than 2^-119 of it are lost
    return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-y));
}

}  // namespace dmoe
