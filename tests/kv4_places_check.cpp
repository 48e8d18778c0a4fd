// Checks the token places of the attention kernels over the 4-bit cache
// (drama3-studio_amd/csrc/kv4_places.hpp) against 64-bit arithmetic, for every
// block that a kernel asks for: up to two behind the last of a sequence.
// Built with g++ and run by test_kv4.py.
#include <algorithm>
#include <cstdio>

#include "kv4_places.hpp"

int main() {
    const int64_t most = INT32_MAX;
    int checked = 0;
    for (const int64_t end : {(int64_t)1, (int64_t)2, (int64_t)63, (int64_t)64, (int64_t)65, (int64_t)4096, (int64_t)100001,
                              most - 200, most - 191, most - 128, most - 127, most - 65, most - 64, most - 63, most - 1, most}) {
        const int64_t last = (end - 1) / dmoe::kKv4Block;
        for (int64_t block = std::max<int64_t>(0, last - 3); block <= last + 2; ++block)
            for (int64_t at = 0; at < dmoe::kKv4Block; ++at, ++checked) {
                const int64_t token = std::min(block * dmoe::kKv4Block + at, end - 1);
                const int64_t left = end - block * dmoe::kKv4Block - at;
                if (dmoe::kv4_token((int)block, (int)at, (int)end) != token || dmoe::kv4_left((int)block, (int)at, (int)end) != left) {
                    std::printf("differ: end %lld block %lld at %lld: token %d, left %d\n", (long long)end, (long long)block,
                                (long long)at, dmoe::kv4_token((int)block, (int)at, (int)end), dmoe::kv4_left((int)block, (int)at, (int)end));
                    return 1;
                }
            }
    }
    std::printf("ok %d\n", checked);
    return 0;
}
