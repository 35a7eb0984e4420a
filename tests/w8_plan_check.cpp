// The plan of an 8-bit projection and of the kernel over a shared prefix
// (csrc/tl_serving.h) on the CPU: every tile of results is taken once, what a workgroup
// reads lies in the packed weights and the scratch, and a workgroup's LDS fits; every
// key of a row is some tile's.
#include <cstdio>
#include <vector>

#include "tl_serving.h"

using namespace tl;

static int wrong;
#define CHECK(c)                                                                                        \
    do {                                                                                                \
        if (!(c) && ++wrong < 20) std::printf("line %d, m %d n %d k %d glu %d: %s\n", __LINE__, m, n, k, glu, #c); \
    } while (0)

static int kinds[8], shapes_seen[W8_SHAPES];

static void one(int m, int n, int k, bool glu) {
    const W8Plan p = w8_plan(m, n, k, glu);
    const int blocks = w8_blocks(k), tiles = w8_tiles(n, glu), mbs = (m + 15) / 16;
    kinds[p.kind]++;
    CHECK(blocks % 2 == 0 && blocks * 64 >= k && (blocks - 2) * 64 < k);
    CHECK(tiles * 16 >= n * (glu ? 2 : 1));
    CHECK(w8_packed_bytes(n, k, glu) == (int64_t)tiles * blocks * 1024 + tiles * 16ll * 4);
    CHECK(p.lds <= kW8Lds);
    CHECK(p.grid_x >= 1 && p.grid_y >= 1 && p.grid_y <= 65535);
    if (p.kind == W8_ROW) {
        CHECK(m <= 4 && w8_scratch(m, k) == 0 && w8_slots(m, k) <= kW8Slots);
        CHECK(p.split == 1 || p.split == 2 || p.split == 4 || p.split == 8);
        const int per = kW8Waves / p.split, units = (n + 15) / 16;
        CHECK((int64_t)p.grid_x * per >= units && (int64_t)(p.grid_x - 1) * per < units);
        CHECK(p.lds >= (int64_t)blocks * 64 * m + kW8Waves * (glu ? 2 : 1) * 1024);
        // the threads hold every unit of every row
        CHECK((int64_t)w8_slots(1, k) * kW8Threads >= blocks * 8);
        return;
    }
    CHECK((int64_t)w8_scratch(m, k) == w8_rows_off(m) + (int64_t)mbs * blocks * 1024 && w8_rows_off(m) >= 4ll * m);
    CHECK(w8_rows_off(m) % 1024 == 0);
    CHECK(p.quant_waves == 1 || p.quant_waves == 2 || p.quant_waves == 4 || p.quant_waves == 8);
    if (p.kind == W8_SPLIT) {
        CHECK((int64_t)p.grid_x * p.nt >= tiles && (int64_t)(p.grid_x - 1) * p.nt < tiles);
        CHECK(p.grid_y * p.mt >= mbs && (p.grid_y - 1) * p.mt < mbs);
        CHECK(!glu || p.nt % 2 == 0);
        CHECK(p.nt * p.mt * 1024 <= 65536);
        return;
    }
    const int sn = kW8Sides[p.shape][0], sm = kW8Sides[p.shape][1];
    CHECK((int64_t)p.tiles.n * sn >= tiles && (int64_t)(p.tiles.n - 1) * sn < tiles);
    CHECK((int64_t)p.tiles.m * sm >= mbs && (int64_t)(p.tiles.m - 1) * sm < mbs);
    CHECK(!glu || p.shape != W8_14x16);
    shapes_seen[p.shape]++;
    CHECK((int64_t)p.grid_x == (int64_t)p.tiles.n * p.tiles.m);
    CHECK((int64_t)p.grid_x * 512 < 1ll << 32);
    if (p.grid_x > 3000000) return;
    std::vector<char> seen(p.grid_x);
    for (int b = 0; b < p.grid_x; b++) {
        int tn = -1, tm = -1;
        p.tiles.tile(b, tn, tm);
        CHECK(tn >= 0 && tn < p.tiles.n && tm >= 0 && tm < p.tiles.m);
        if (tn < 0 || tn >= p.tiles.n || tm < 0 || tm >= p.tiles.m) return;
        CHECK(!seen[(size_t)tm * p.tiles.n + tn]);
        seen[(size_t)tm * p.tiles.n + tn] = 1;
    }
}

static void prefix(int rows, int heads, int n_kv, int len) {
    const int m = rows, n = heads, k = len, glu = n_kv;
    const PrefixPlan p = prefix_plan(rows, heads, n_kv, len);
    const int64_t columns = (int64_t)rows * (heads / n_kv);
    CHECK(p.qw == 1 || p.qw == 4);
    CHECK((int64_t)p.qblocks * 32 * p.qw >= columns && (int64_t)(p.qblocks - 1) * 32 * p.qw < columns);
    CHECK(p.splits >= 1 && p.splits <= len && (int64_t)p.grid == (int64_t)p.qblocks * n_kv * p.splits);
    CHECK((int64_t)p.grid * 256 < 1ll << 32);
    // the workgroups of both kinds, each once
    if (p.grid > 100000) return;
    for (int own : {1, 7, 255, 256, 257, 512}) {
        const SharedRoles roles{p.grid, own};
        std::vector<char> seen(p.grid + own);
        for (int b = 0; b < p.grid + own; b++) {
            int at = -1;
            const bool mine = roles.is_own(b, at);
            CHECK(at >= 0 && at < (mine ? own : p.grid));
            if (at < 0 || at >= (mine ? own : p.grid)) return;
            CHECK(!seen[mine ? p.grid + at : at]);
            seen[mine ? p.grid + at : at] = 1;
        }
    }
    for (int side : {8, 16})
        for (int own : {1, 512}) {
            const int lanes = shared_join_lanes(side, p.splits, own, (int64_t)rows * heads);
            CHECK(lanes >= 1 && lanes <= side && side % lanes == 0);
        }
}

static void rows_behind(int len, int pos) {
    const int m = len, n = pos, k = 0, glu = 0;
    const int tiles = shared_tiles(len, pos);
    CHECK(tiles >= 1);
    if (pos < 0) {
        CHECK(tiles == 1 && !shared_adds(len, pos));
        return;
    }
    const int first = shared_adds(len, pos) ? len : 0, base = first & ~31, end = pos + 1;
    CHECK(shared_adds(len, pos) == (end >= len));
    if (end > first) CHECK(base <= first && first < base + kPagedTile && (int64_t)base + (int64_t)tiles * kPagedTile >= end &&
                           (int64_t)base + (int64_t)(tiles - 1) * kPagedTile < end);
    else CHECK(tiles == 1);
}

int main() {
    const int shapes[][2] = {{1, 1}, {15, 17}, {16, 64}, {17, 63}, {33, 77}, {100, 4096}, {300, 129}, {2048, 2048}, {2048, 5632},
                             {2560, 2048}, {5632, 2048}, {6144, 4096}, {8000, 2048}, {8192, 8192}, {14336, 4096}, {32000, 2048},
                             {64, 1 << 17}, {100003, 100}, {1 << 20, 64}};
    const int rows[] = {1, 2, 3, 4, 5, 7, 8, 15, 16, 17, 31, 32, 33, 48, 49, 64, 65, 100, 128, 200, 255, 256, 257, 300, 512,
                        1000, 2001, 4096, 8192, 65537, 1 << 17};
    for (auto& s : shapes)
        for (int m : rows)
            for (int glu = 0; glu < 2; glu++)
                if ((int64_t)m * s[0] < 1ll << 38) one(m, s[0], s[1], glu);
    const int m = 0, n = 0, k = 0, glu = 0;
    for (int kind = W8_ROW; kind <= W8_TILE; kind++) CHECK(kinds[kind] > 5);
    for (int shape = 0; shape < W8_SHAPES; shape++) CHECK(shapes_seen[shape] > 0);
    const int heads[][2] = {{32, 4}, {8, 8}, {5, 1}, {40, 8}, {1, 1}, {128, 1}, {1024, 1024}};
    for (auto& h : heads)
        for (int r : {1, 2, 3, 8, 16, 17, 33, 64, 257, 4096, 1 << 20})
            for (int len : {1, 31, 255, 256, 257, 1000, 65536, 1 << 30})
                if ((int64_t)r * h[0] < 1 << 30) prefix(r, h[0], h[1], len);
    for (int len : {1, 7, 8, 31, 32, 33, 127, 128, 129, 1000, 4096})
        for (int pos = -2; pos < len + 700; pos++) rows_behind(len, pos);
    rows_behind(1 << 29, (1 << 30) - 1);
    rows_behind(1 << 30, (1 << 30) - 1);
    std::printf("%d wrong\n", wrong);
    return wrong ? 1 : 0;
}
