// Places of tokens in a sequence of the 4-bit cache: plain C++, shared by the
// attention kernels and a g++-built check.
#pragma once

#include <stdint.h>

namespace dmoe {

constexpr int kKv4Block = 64;  // tokens an attention step takes

// Token `at` of a block, or the last of `end` tokens if that comes first.
// Loads are sent ahead, for blocks up to two behind the last: with the most
// tokens that a length can name, 2^31 - 1, such a block's tokens do not fit 31
// bits, but 32.
constexpr int kv4_token(int block, int at, int end) {
    const uint32_t token = (uint32_t)block * kKv4Block + (uint32_t)at, last = (uint32_t)end - 1;
    return (int)(token < last ? token : last);
}

// How many of a block's tokens from `at` on there are of `end` (none: zero or less).
constexpr int kv4_left(int block, int at, int end) {
    return (int)((uint32_t)end - (uint32_t)block * kKv4Block - (uint32_t)at);
}

}  // namespace dmoe
