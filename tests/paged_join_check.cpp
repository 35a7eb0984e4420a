// Which workgroups of the joining kernel join what (csrc/tl_serving.h), on the CPU:
// every (row, head block) whose tiles several workgroups had is joined at exactly one
// boundary between their runs, no other is, and the grid does not grow with the rows.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "tl_serving.h"

using namespace tl;

static int wrong;
#define CHECK(c)                                              \
    do {                                                      \
        if (!(c) && ++wrong < 20) std::printf("line %d: %s\n", __LINE__, #c); \
    } while (0)

int main() {
    srand(3);
    long split = 0;
    for (int round = 0; round < 4000; round++) {
        const int workgroups = 1 + rand() % (round % 2 ? 600 : 12), longest = 1 + rand() % (round % 3 ? 40 : 400);
        std::vector<int32_t> starts;   // of the units, and their end
        int32_t tiles = 0;
        for (int units = 1 + rand() % 300; units > 0; units--) {
            starts.push_back(tiles);
            tiles += 1 + rand() % longest;
        }
        starts.push_back(tiles);
        const PagedShare s = paged_share(tiles, workgroups);
        std::vector<int> joined(starts.size(), 0);
        for (int32_t w = 1; w < workgroups; w++) {
            if (s.start(w) >= tiles || s.start(w) == s.start(w - 1)) continue;   // as the kernel leaves
            const size_t u = std::upper_bound(starts.begin(), starts.end(), s.start(w)) - starts.begin() - 1;
            joined[u] += paged_joins_at(s, w, starts[u]);
        }
        for (size_t u = 0; u + 1 < starts.size(); u++) {
            const bool several = s.owner(starts[u]) != s.owner(starts[u + 1] - 1);
            CHECK(joined[u] == several);
            split += several;
        }
    }
    CHECK(split > 10000);
    const PagedJoinGrid few = paged_join_grid(64, 32, 4, 512), many = paged_join_grid((1 << 24) - 1, 32, 4, 512),
                        alone = paged_join_grid(65, 12, 12, 512), wide = paged_join_grid(100, 48, 4, 512);
    CHECK(few.x == 64 && few.y == 32);
    CHECK(many.x == 511 && many.y == 8);
    CHECK(alone.x == 511 && alone.y == 1 && wide.y == 8);
    std::printf("%d wrong\n", wrong);
    return wrong ? 1 : 0;
}
