// The plan of a 4-bit projection (csrc/tl_serving.h) against the scratch that a caller
// gives it, on the CPU: whatever the rows and the weights' shape, the digits that any
// workgroup reads lie inside w4_scratch() bytes, every row block is taken, and a
// workgroup's LDS fits.
#include <cstdio>

#include "tl_serving.h"

using namespace tl;

static int wrong;
static long spare;   // workgroup rows with row blocks to spare
#define CHECK(c)                                                                                          \
    do {                                                                                                  \
        if (!(c) && ++wrong < 20) std::printf("line %d, m %d n %d k %d group %d: %s\n", __LINE__, m, n, k, group, #c); \
    } while (0)

static void one(int m, int n, int k, int group) {
    const W4Plan p = w4_plan(m, n, k, group);
    const int cbs = w4_row_blocks(m);
    CHECK(p.cb == 1 || p.cb == 2 || p.cb == 4);
    CHECK(p.split == 1 || p.split == 2 || p.split == 4 || p.split == 8);
    CHECK(p.lds > 0 && p.lds <= kW4Lds);
    CHECK((int64_t)p.grid_x * (kW4Waves / p.split) >= w4_tiles(n) && (int64_t)(p.grid_x - 1) * (kW4Waves / p.split) < w4_tiles(n));
    CHECK(p.grid_y >= 1 && p.grid_y <= 65535 && p.grid_y * p.cb >= cbs && (p.grid_y - 1) * p.cb < cbs);
    if (p.convert) {
        CHECK(m <= 4 && p.cb == 1 && p.grid_y == 1 && 4 * m <= p.cols && w4_slots(m, k) <= kW4Slots);
        return;
    }
    CHECK(p.cols == 16);
    const int64_t scratch = (int64_t)w4_scratch(m, k);
    CHECK(w4_bexp_off(m) >= 4ll * m && w4_bexp_off(m) % 16 == 0 && w4_digit_off(m, k) % 16 == 0);
    spare += p.grid_y * p.cb != cbs;
    // the workgroup rows at both ends, every row block of theirs
    for (int y : {0, p.grid_y - 2, p.grid_y - 1})
        for (int c = 0; c < p.cb && y >= 0; c++) {
            const int b = w4_row_block(y, p.cb, c, m);
            CHECK(b >= 0 && b < cbs && (b == y * p.cb + c || y * p.cb + c >= cbs));
            CHECK(w4_bexp_off(m) + (b + 1) * w4_bexp_bytes(k) <= w4_digit_off(m, k));
            CHECK(w4_digit_off(m, k) + (b + 1) * w4_frag_bytes(k, 16) <= scratch);
        }
}

int main() {
    const int shapes[][2] = {{1, 32}, {16, 128}, {17, 96}, {200, 1024}, {300, 2112}, {2048, 2048}, {2048, 5632}, {2560, 2048},
                             {5632, 2048}, {8000, 2048}, {8192, 8192}, {14336, 8192}, {16400, 2080}, {32000, 2048}, {32000, 512},
                             {40, 16416}, {24, 32768}, {50, 20480}, {128256, 8192}, {1 << 24, 1024}};
    const int many[] = {100, 127, 255, 256, 300, 333, 513, 2048, 4097, 65535, 1 << 17};
    for (auto& s : shapes)
        for (int group : {32, 64, 128}) {
            if (s[1] % group || s[1] / group > kW4MaxGroups) continue;
            for (int m = 1; m <= 80; m++) one(m, s[0], s[1], group);
            for (int m : many) one(m, s[0], s[1], group);
        }
    const int m = 0, n = 0, k = 0, group = 0;
    one(3, 20, 131072, 128);
    one(9, 20, 131072, 128);
    // the quantizer's launch, at the most weights there may be
    for (int64_t units : {1ll, 256ll, 257ll, 1ll << 31, (1ll << 32) - 255, (1ll << 32) - 4}) {
        CHECK(w4_quantize_grid(units) >= 1 && (uint64_t)w4_quantize_grid(units) * 256 < 1ull << 32);
        CHECK(units > 1 << 30 || (int64_t)w4_quantize_grid(units) * 256 >= units);
    }
    CHECK(spare > 100);   // the case is among them
    std::printf("%d wrong\n", wrong);
    return wrong ? 1 : 0;
}
