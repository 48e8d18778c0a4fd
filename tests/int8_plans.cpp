// Prints the plan (shape, shares of K) of each product "rows n k gated" on its input.
#include <cstdio>

#include "int8.hpp"

int main() {
    int rows, n, k, gated;
    while (std::scanf("%d %d %d %d", &rows, &n, &k, &gated) == 4) {
        const dmoe::Int8Plan p = dmoe::int8_plan(rows, n, k, gated != 0);
        std::printf("%d %d\n", (int)p.shape, p.splits);
    }
}
