// Index arithmetic of the paged cache (csrc/tl_serving.h) on the CPU: every table
// lookup stays in the table, every row in its page and every page in the pool,
// whatever the table holds; the workgroups' shares tile the keys.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "tl_serving.h"

using namespace tl;

static int wrong;
#define CHECK(c)                                              \
    do {                                                      \
        if (!(c)) {                                           \
            wrong++;                                          \
            if (wrong < 20) std::printf("line %d: %s\n", __LINE__, #c); \
        }                                                     \
    } while (0)

int main() {
    srand(1);
    for (int shift = 3; shift <= 10; shift++) {
        const int seqs = 3, max_pages = 5, n_pages = 7, n_kv = 3, hd = 64;
        std::vector<int32_t> table(seqs * 9);
        for (auto& e : table) e = rand() % 4 ? rand() % n_pages : (rand() % 2 ? -1 - rand() % 100 : n_pages + rand() % 1000);
        table[4] = INT32_MIN;
        table[5] = INT32_MAX;
        PagedGeom g{table.data(), 9, (int64_t)n_kv * hd << shift, seqs, max_pages, n_pages, shift, n_kv, hd};
        std::set<int64_t> seen;
        for (int s = -2; s < seqs + 2; s++)
            for (int64_t p = -2; p < ((int64_t)max_pages << shift) + 2; p++) {
                const PagedRow k = paged_row_kind(g, s, (int32_t)p);
                CHECK((k == PAGED_ROW_PADDING) == (s < 0));
                CHECK((k == PAGED_ROW_FAULT) == (s >= seqs || (s >= 0 && p >= ((int64_t)max_pages << shift))));
                if (k != PAGED_ROW_OK || p < 0) continue;
                const int32_t e = table[s * 9 + (p >> shift)];
                const int32_t page = paged_page(g, s, (int32_t)p);
                CHECK(page == (e >= 0 && e < n_pages ? e : -1));
                if (page < 0) continue;
                for (int h = 0; h < n_kv; h++) {
                    const int64_t at = paged_row(g, page, h, (int32_t)p);
                    CHECK(at >= page * g.page_stride && at + hd <= (page + 1) * g.page_stride && at % hd == 0);
                    CHECK(at == page * g.page_stride + ((int64_t)h * (1 << shift) + p % (1 << shift)) * hd);
                }
            }
    }
    // offsets past 2^31 elements and past 2^32 bytes
    {
        int32_t entry = 999999;
        PagedGeom g{&entry, 1, (int64_t)8 * 1024 * 128, 1, 1, 1000000, 10, 8, 128};
        CHECK(paged_page(g, 0, 1023) == 999999);
        CHECK(paged_row(g, 999999, 7, 1023) == 999999ll * 1048576 + (7ll * 1024 + 1023) * 128);
        CHECK(paged_row_kind(g, 0, INT32_MAX) == PAGED_ROW_FAULT);
        g.max_pages = 1 << 20;
        CHECK(paged_row_kind(g, 0, (1 << 30) - 1) == PAGED_ROW_OK && paged_row_kind(g, 0, 1 << 30) == PAGED_ROW_FAULT);
    }
    // shares: every tile has one owner, runs follow one another and differ by at most one; a workgroup leaves
    // at most one part in each of its two places
    for (int w : {1, 2, 3, 7, 64, 255, 768})
        for (int64_t tiles : {1ll, 2ll, 63ll, 64ll, 65ll, 767ll, 768ll, 769ll, 5000ll, (1ll << 31) - 1}) {
            const PagedShare s = paged_share((int32_t)tiles, w);
            CHECK(s.start(0) == 0 && s.start(w) == tiles);
            for (int i = 0; i < w; i++) {
                const int64_t n = s.start(i + 1) - s.start(i);
                CHECK(n == s.per || n == s.per + 1);
                if (n == 0) continue;
                CHECK(s.owner(s.start(i)) == i && s.owner(s.start(i + 1) - 1) == i);
            }
            if (tiles > 5000) continue;
            srand(w);
            std::set<int> parts;
            for (int64_t unit = 0; unit < tiles;) {
                const int64_t end = std::min<int64_t>(tiles, unit + 1 + rand() % 40);
                const int w0 = s.owner(unit), w1 = s.owner(end - 1);
                for (int i = w0; i <= w1 && w0 != w1; i++) {
                    const int p = paged_part(s, i, unit);
                    CHECK(p / 2 == i && parts.insert(p).second);
                }
                unit = end;
            }
        }
    CHECK(paged_tiles(-3) == 1 && paged_tiles(0) == 1 && paged_tiles(1) == 1 && paged_tiles(128) == 1 && paged_tiles(129) == 2);
    CHECK(paged_tiles(1 << 30) == 1 << 23);
    PagedGeom g{};
    g.max_pages = 1 << 20;
    g.page_shift = 10;
    CHECK(paged_countable(g, 1, 255) && paged_countable(g, 255, 1) && !paged_countable(g, 256, 1) && !paged_countable(g, 2, 128));
    g.max_pages = 1;
    CHECK(paged_countable(g, 1 << 20, 100) && !paged_countable(g, 1 << 20, 1 << 9));
    // rows that share no byte, against the bytes themselves
    srand(5);
    for (int i = 0; i < 200000; i++) {
        const int64_t rows = rand() % 4, wp = 1 + rand() % 6, wq = 1 + rand() % 6, sp = wp + rand() % 9;
        const int64_t sq = rand() % 2 && sp >= wq ? sp : wq + rand() % 9, at = rand() % 70;
        char bytes[256] = {};
        const char *p = bytes + 64, *q = bytes + 30 + at;
        bool apart = true;
        for (int64_t r = 0; r < rows; r++) for (int64_t b = 0; b < wp; b++) bytes[64 + r * sp + b] = 1;
        for (int64_t r = 0; r < rows; r++) for (int64_t b = 0; b < wq; b++) apart &= !q[r * sq + b];
        const bool said = rows_apart(p, sp, wp, q, sq, wq, rows);
        CHECK(!said || apart);
        if (rows <= 1) CHECK(said == apart);
        // side by side within each row
        if (sp == sq && q >= p + wp && q + wq <= p + sp) CHECK(said);
    }
    std::printf("%d wrong\n", wrong);
    return wrong ? 1 : 0;
}
