// The plans of 8-bit projections (csrc/tl_serving.h): for each "m n k gated" on the input a line
// "kind split nt mt shape blocks slots_of_a_row".
#include <cstdio>

#include "tl_serving.h"

int main() {
    int m, n, k, gated;
    while (std::scanf("%d %d %d %d", &m, &n, &k, &gated) == 4) {
        const tl::W8Plan p = tl::w8_plan(m, n, k, gated != 0);
        std::printf("%d %d %d %d %d %d %d\n", p.kind, p.split, p.nt, p.mt, p.shape, tl::w8_blocks(k), tl::w8_slots(1, k));
    }
}
