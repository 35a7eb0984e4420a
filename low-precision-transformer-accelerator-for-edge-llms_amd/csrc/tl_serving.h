// tl_serving.h -- declarations of the serving operators (paged KV cache, 4-bit and 8-bit
// projections, token log probabilities), shared by their kernels (tl_paged.hip,
// tl_prefix.hip, tl_w4.hip, tl_w8.hip, tl_score.hip) and the C++ runtime (tl_runtime.hip).  The index
// arithmetic at the top is host code too: a CPU test compiles it by itself.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

#if defined(__HIPCC__)
#define TL_HD __host__ __device__
#else
#define TL_HD
#endif

namespace tl {

// The geometry of a paged cache: position t of sequence s lies in page
// table[s][t / page_size], at row t % page_size of each KV head's block of that
// page.  page_size is a power of two, at least 8.
struct PagedGeom {
    const int32_t* table;   // [n_seqs][table_stride]
    int64_t table_stride;
    int64_t page_stride;    // elements between pages
    int32_t n_seqs, max_pages, n_pages;
    int32_t page_shift;     // log2(page_size)
    int32_t n_kv, head_dim;
};

// the page that holds position pos (0 <= pos < max_pages * page_size) of
// sequence seq (0 <= seq < n_seqs), or -1 where the table's entry names none
TL_HD inline int32_t paged_page(const PagedGeom& g, int32_t seq, int32_t pos) {
    const int32_t p = g.table[(int64_t)seq * g.table_stride + (pos >> g.page_shift)];
    return p >= 0 && p < g.n_pages ? p : -1;
}

// elements from the cache's base to row pos of KV head `head` in `page`: 64
// bits, as a cache may hold more than 2^31 elements
TL_HD inline int64_t paged_row(const PagedGeom& g, int32_t page, int32_t head, int32_t pos) {
    const int32_t at = pos & ((1 << g.page_shift) - 1);
    return (int64_t)page * g.page_stride + (((int64_t)head << g.page_shift) + at) * g.head_dim;
}

// What a row of an append or attention call names.  A row of a padded batch has
// a negative sequence and is left alone; a row whose sequence or position lies
// outside the cache is a fault and is left alone too.
enum PagedRow : int { PAGED_ROW_OK = 0, PAGED_ROW_PADDING = 1, PAGED_ROW_FAULT = 2 };
TL_HD inline PagedRow paged_row_kind(const PagedGeom& g, int32_t seq, int32_t pos) {
    if (seq < 0) return PAGED_ROW_PADDING;
    if (seq >= g.n_seqs) return PAGED_ROW_FAULT;
    return pos < ((int64_t)g.max_pages << g.page_shift) ? PAGED_ROW_OK : PAGED_ROW_FAULT;
}

// Attention shares out tiles of kPagedTile keys.  Row r has paged_tiles(n) of them
// for each of its head blocks (a row without keys one, for its zeros); all tiles
// of a call, in the order row, head block, key, are dealt to the workgroups in
// runs that differ in length by at most one, whatever the rows' lengths are.
constexpr int32_t kPagedTile = 128;
TL_HD inline int32_t paged_tiles(int32_t n) { return n > 0 ? (int32_t)(((int64_t)n + kPagedTile - 1) / kPagedTile) : 1; }

struct PagedShare {
    int32_t per;   // tiles of every workgroup
    int32_t rem;   // the first rem have one more
    TL_HD int32_t start(int32_t w) const { return w * per + (w < rem ? w : rem); }
    TL_HD int32_t owner(int32_t tile) const {
        const int32_t longer = rem * (per + 1);
        return tile < longer ? (int32_t)((uint32_t)tile / (uint32_t)(per + 1))
                             : rem + (int32_t)((uint32_t)(tile - longer) / (uint32_t)per);
    }
};
TL_HD inline PagedShare paged_share(int32_t tiles, int32_t workgroups) {
    const int32_t per = (int32_t)((uint32_t)tiles / (uint32_t)workgroups);
    return PagedShare{per, tiles - per * workgroups};
}
// A workgroup leaves at most two parts of rows that others share with it: one at
// the start of its run (0) and one at the end (1).
TL_HD inline int32_t paged_part(const PagedShare& s, int32_t w, int32_t unit_start) {
    return 2 * w + (unit_start > s.start(w) ? 1 : 0);
}
// Whether the parts of the unit (row, head block) that starts at tile `unit` and holds
// tile start(w) are joined at the boundary in front of workgroup w's run: of a unit's
// boundaries, the first inside it.  Units that one workgroup has whole have none.
TL_HD inline bool paged_joins_at(const PagedShare& s, int32_t w, int32_t unit) {
    return s.start(w) > unit && s.start(w - 1) <= unit;
}
// Rows that share the first `len` positions of one sequence.  A row at pos from len - 1 on
// adds the parts that the prefix's kernel left to its own keys, len .. pos, whose tiles
// count from the last multiple of 32 up to len; a row before that is a row of the prefix's
// sequence at pos and has all its keys from there.
TL_HD inline bool shared_adds(int32_t len, int32_t pos) { return pos >= 0 && pos + 1 >= len; }
TL_HD inline int32_t shared_tiles(int32_t len, int32_t pos) {
    if (!shared_adds(len, pos)) return paged_tiles(pos + 1);
    return paged_tiles(pos + 1 > len ? pos + 1 - (len & ~31) : 0);
}

// The kernel over a shared prefix: workgroups of 32 qw columns (rows times the query heads
// of a KV head), the keys of each split so that the whole GPU has some.
struct PrefixPlan {
    int32_t qw;        // 1 or 4
    int32_t qblocks;   // column blocks
    int32_t splits;
    int32_t grid;
};
// Two workgroups to a CU where each still has 2048 keys (64 rows over 131072 keys of 8 heads
// of 128 259 us, one to a CU 311), else one, which leaves half the parts (8 rows over 16000
// keys of 8 heads of 64 16.3 us and 20.2), each of one or four tiles' keys at least (4 rows over
// 500 keys 11.6 us, with 256 keys each 12.4; 32 rows over 1536 17.1, with 128 18.1).
constexpr int32_t kPrefixWorkgroups = 256;
constexpr int64_t kPrefixManyKeys = 2048;
TL_HD inline int32_t prefix_split_keys(int32_t qw) { return qw == 1 ? 128 : 256; }
inline PrefixPlan prefix_plan(int32_t rows, int32_t n_heads, int32_t n_kv, int32_t len) {
    const int64_t columns = (int64_t)rows * (n_heads / n_kv);
    PrefixPlan p;
    p.qw = columns <= 64 ? 1 : 4;
    p.qblocks = (int32_t)((columns + 32 * p.qw - 1) / (32 * p.qw));
    const int64_t units = (int64_t)p.qblocks * n_kv;
    const int32_t least = prefix_split_keys(p.qw);
    const int64_t most = ((int64_t)len + least - 1) / least, all = (int64_t)len * units >= 2 * kPrefixWorkgroups * kPrefixManyKeys ? 2 * kPrefixWorkgroups : kPrefixWorkgroups,
                  want = (all + units - 1) / units;
    p.splits = (int32_t)(want < most ? want : most);
    if (p.splits < 1) p.splits = 1;
    p.grid = (int32_t)(units * p.splits);
    return p;
}

// Which workgroups of the kernel of a shared prefix take its keys and which the rows' own:
// they take turns 256 at a time, one of each on every CU, as the ones multiply while the
// others wait for memory; what is left of either kind follows.
struct SharedRoles {
    int32_t prefix, own;   // workgroups of each kind
    TL_HD bool is_own(int32_t b, int32_t& at) const {
        const int32_t k = (prefix < own ? prefix : own) >> 8;
        if (b < k << 9) {
            at = (b >> 9 << 8) + (b & 255);
            return b >> 8 & 1;
        }
        at = b - (k << 8);
        if (at < prefix) return false;
        at = b - prefix;
        return true;
    }
};

// Parts of a query head that the join takes side by side, of the `side` that a workgroup can:
// about four to each thread (the prefix's splits and what the own keys may be split into).
inline int32_t shared_join_lanes(int32_t side, int32_t splits, int32_t own_workgroups, int64_t heads) {
    const int64_t parts = splits + 1 + 8 * (int64_t)own_workgroups / (heads > 0 ? heads : 1);
    int32_t lanes = 1;
    while (lanes < side && 4 * lanes < parts) lanes *= 2;
    return lanes;
}

// The joining kernel's workgroups.  Up to 64 rows it has one per row and head; more
// rows than that each would have to be looked for, though only workgroups - 1 (row, head
// block)s can be split, so there it has one per boundary and head of a block.
constexpr int32_t kPagedFewRows = 64;
struct PagedJoinGrid {
    int32_t x, y;
};
inline PagedJoinGrid paged_join_grid(int32_t rows, int32_t n_heads, int32_t n_kv, int32_t workgroups) {
    if (rows <= kPagedFewRows) return {rows, n_heads};
    const int32_t rep = n_heads / n_kv;
    return {workgroups - 1, rep < 8 ? rep : 8};
}
// whether a call's tiles can be counted in 31 bits, were every row as long as the
// table allows
inline bool paged_countable(const PagedGeom& g, int32_t rows, int32_t head_blocks) {
    const int64_t most = paged_tiles((int32_t)((int64_t)g.max_pages << g.page_shift));
    return most * head_blocks <= INT32_MAX / (rows > 0 ? rows : 1);
}

// Whether two sets of rows (bytes: strides s, widths w) share no byte: one behind the
// other, or, with one stride, side by side in each row of a wider matrix.
inline bool rows_apart(const void* p, int64_t sp, int64_t wp, const void* q, int64_t sq, int64_t wq, int64_t rows) {
    if (rows <= 0) return true;
    const int64_t d = (int64_t)((uintptr_t)q - (uintptr_t)p);   // of q's rows from p's
    if (d >= (rows - 1) * sp + wp || -d >= (rows - 1) * sq + wq) return true;
    if (rows == 1 || sp != sq || sp <= 0) return false;
    const int64_t at = (d % sp + sp) % sp;
    return at >= wp && at + wq <= sp;
}

// Projections with 4-bit weights: sizes, the plan of a call, and where its pieces lie.
//
// Weights come in tiles of 16 rows and blocks of 128 columns.  Scratch of a call
// (w4_scratch() bytes): the exponents of its rows of x; of each four rows ("row block")
// the exponents of their blocks, w4_bexp_bytes(k) bytes; then the row blocks' digits,
// w4_frag_bytes(k, 16) bytes each.
constexpr int32_t kW4Waves = 8, kW4Threads = 64 * kW4Waves;
constexpr int32_t kW4MaxGroups = 1024;
constexpr int64_t kW4EnoughWaves = 1024;
constexpr int64_t kW4Lds = 152 * 1024;   // of a workgroup's 160 KiB
constexpr int32_t kW4Slots = 4;          // units of 8 columns of x that a thread keeps in registers
constexpr int32_t kW4Chunk = 8;          // blocks of 128 columns whose digits are in LDS at a time

TL_HD inline int32_t w4_blocks(int32_t k) { return (k + 127) / 128; }
TL_HD inline int32_t w4_tiles(int32_t n) { return (n + 15) / 16; }
TL_HD inline int32_t w4_row_blocks(int32_t m) { return (m + 3) / 4; }
TL_HD inline int32_t w4_groups(int32_t k, int32_t group) { return w4_blocks(k) * (128 / group); }   // with the padding's
TL_HD inline int64_t w4_frag_bytes(int32_t k, int32_t cols) { return (int64_t)w4_blocks(k) * 128 * cols; }
TL_HD inline int64_t w4_bexp_bytes(int32_t k) { return (int64_t)w4_blocks(k) * 8; }   // int16 [block][row]
TL_HD inline int64_t w4_bexp_off(int32_t m) { return ((int64_t)m * 4 + 15) / 16 * 16; }
TL_HD inline int64_t w4_digit_off(int32_t m, int32_t k) {
    return w4_bexp_off(m) + (w4_row_blocks(m) * w4_bexp_bytes(k) + 15) / 16 * 16;
}
// units of all of `rows` rows that a thread takes
TL_HD inline int32_t w4_slots(int32_t rows, int32_t k) { return rows * ((w4_blocks(k) * 16 + kW4Threads - 1) / kW4Threads); }
// The row block that workgroup row y takes as its c-th of cb.  Where cb does not divide
// the row blocks, the last workgroup row has some to spare: they stand for the last one
// again, and their results go nowhere.
TL_HD inline int32_t w4_row_block(int32_t y, int32_t cb, int32_t c, int32_t m) {
    const int32_t b = y * cb + c, last = w4_row_blocks(m) - 1;
    return b < last ? b : last;
}
inline size_t w4_scratch(int32_t m, int32_t k) {
    return m <= 0 ? 0 : (size_t)(w4_digit_off(m, k) + w4_row_blocks(m) * w4_frag_bytes(k, 16));
}

// workgroups of 256 threads that quantize units of 8 weights: a launch holds fewer than
// 2^32 threads, which 2^35 weights would be
inline uint32_t w4_quantize_grid(int64_t units) {
    const int64_t all = (units + 255) / 256;
    return (uint32_t)(all < 1 << 23 ? all : 1 << 23);
}

struct W4Plan {
    bool convert;          // one kernel that turns x into digits itself (up to four rows)
    int32_t cb;            // row blocks of a workgroup: 1, 2 or 4
    int32_t split;         // wavefronts that share a tile of 16 weight rows: 1, 2, 4 or 8
    int32_t cols;          // columns of a product in use by the digits' layout
    int32_t grid_x, grid_y;
    int64_t lds;           // bytes of a workgroup
};

// LDS of a workgroup: scales, sums, exponents, a word per row and block, digits
inline int64_t w4_lds(int32_t k, int32_t group, int32_t split, int32_t cb, int64_t digits) {
    return (int64_t)(kW4Waves / split) * w4_groups(k, group) * 64 + kW4Waves * 16 * 4 * cb * 4 + 192 +
           cb * w4_blocks(k) * 16 + digits;
}

inline W4Plan w4_plan(int32_t m, int32_t n, int32_t k, int32_t group) {
    const int32_t tiles = w4_tiles(n), cbs = w4_row_blocks(m);
    W4Plan p{};
    p.cols = m == 1 ? 4 : m == 2 ? 8 : 16;
    // Up to four rows each workgroup converts them itself where its registers hold them
    // (their digits are 64 KiB then at most): one kernel.  One row by 32000 x 2048: 11.8 us,
    // 18.3 through scratch; by 14336 x 8192: 14.5, 28.3; four by 5632 x 2048: 7.9, 10.3.
    // More rows would be converted by too many: 16 by 5632 x 2048 16.1, 10.7.
    p.convert = cbs == 1 && w4_slots(m, k) <= kW4Slots;
    p.cb = 1;
    int64_t digits;
    if (p.convert) {
        digits = w4_frag_bytes(k, p.cols);
        // wavefronts per tile: enough of them for 4 on each CU (one row by 14336 x 8192
        // 14.5 us, with half of them 19.6; by 5632 x 2048 5.8 in a graph, with half of them
        // 6.3, with twice 6.8; four by 5632 x 2048 7.9, with twice 8.9.  Two rows by 8192 x
        // 8192 would rather have twice: 11.8 us for 14.0)
        p.split = 1;
        while (p.split < kW4Waves && ((int64_t)tiles * p.split < kW4EnoughWaves || w4_lds(k, group, p.split, 1, digits) > kW4Lds))
            p.split *= 2;
    } else {
        p.cols = 16;
        // What a workgroup moves through its CU: 16 CB bytes of digits and 8 of weights per
        // tile and column of x, in as many rounds as 256 CUs need (16 rows by 32000 x 2048:
        // 20.9 us; counted with 512 at once 24.1)
        int64_t best = INT64_MAX;
        digits = 0;
        for (int32_t c : {4, 2, 1}) {
            if (c > 1 && c / 2 >= cbs) continue;   // all of another workgroup row to spare
            const int64_t chunk = (int64_t)2 * c * kW4Chunk * 128 * 16;
            for (int32_t split = 1; split <= kW4Waves; split *= 2) {
                if (w4_lds(k, group, split, c, chunk) > kW4Lds) continue;
                const int32_t per = kW4Waves / split;
                const int64_t wgs = (int64_t)((tiles + per - 1) / per) * ((cbs + c - 1) / c);
                const int64_t cost = (wgs + 255) / 256 * (2 * c + per);
                if (cost < best) {
                    best = cost;
                    p.cb = c;
                    p.split = split;
                    digits = chunk;
                }
            }
        }
    }
    const int32_t per = kW4Waves / p.split;
    p.grid_x = (tiles + per - 1) / per;
    p.grid_y = (cbs + p.cb - 1) / p.cb;
    p.lds = w4_lds(k, group, p.split, p.cb, digits);
    return p;
}

// Projections with 8-bit weights and activations: sizes and the plan of a call.
//
// Weights and quantized rows of x come in tiles of 16 rows and blocks of 64 columns, an
// even number of blocks to a tile.  The tiles of gated weights take turns, gate and up.
// Scratch of a call (w8_scratch() bytes): the scales of its rows, then their blocks.
constexpr int32_t kW8Waves = 8, kW8Threads = 64 * kW8Waves;
constexpr int32_t kW8MaxK = 1 << 17;     // 127 * 128 * 2^17 is below 2^31
constexpr int32_t kW8Slots = 4;          // units of 8 columns of x that a thread keeps in registers
constexpr int32_t kW8Keep = 4;           // and where x is quantized by a kernel of its own
// LDS of a workgroup of single rows: what any launch may have; their columns and the partial
// sums of gated weights take half of it at most
constexpr int64_t kW8Lds = 64 * 1024;
static_assert(kW8Slots * kW8Threads * 8 + kW8Waves * 2 * 1024 <= kW8Lds, "rows and sums fit");

TL_HD inline int32_t w8_blocks(int32_t k) { return (k + 127) / 128 * 2; }
TL_HD inline int32_t w8_tiles(int32_t n, bool glu) { return (n + 15) / 16 * (glu ? 2 : 1); }
TL_HD inline int64_t w8_rows_off(int32_t m) { return ((int64_t)m * 4 + 1023) / 1024 * 1024; }
inline int64_t w8_packed_bytes(int32_t n, int32_t k, bool glu) { return (int64_t)w8_tiles(n, glu) * (w8_blocks(k) * 1024ll + 64); }
// units of all of m rows that a thread takes
TL_HD inline int32_t w8_slots(int32_t m, int32_t k) { return m * ((w8_blocks(k) * 8 + kW8Threads - 1) / kW8Threads); }
TL_HD inline bool w8_in_rows(int32_t m, int32_t k) { return m <= 4 && w8_slots(m, k) <= kW8Slots; }
inline size_t w8_scratch(int32_t m, int32_t k) {
    return m <= 0 || w8_in_rows(m, k) ? 0 : (size_t)(w8_rows_off(m) + (int64_t)((m + 15) / 16) * w8_blocks(k) * 1024);
}

// Which tile a workgroup of the tiled form takes.  Workgroups go to the 8 XCDs in turn, so
// each XCD gets a run of tiles of its own (its L2 then serves a run's operands again), in
// columns of `tall` tiles of tokens.
struct W8Grid {
    int32_t n, m;      // tiles of y
    int32_t tall;
    TL_HD void tile(int32_t b, int32_t& tn, int32_t& tm) const {
        const int32_t all = n * m, per = all / 8, rem = all % 8, xcd = b % 8, at = b / 8;
        const int32_t i = xcd * per + (xcd < rem ? xcd : rem) + at;
        const int32_t group = i / (tall * n), first = group * tall;
        const int32_t h = m - first < tall ? m - first : tall;
        const int32_t in = i - group * tall * n;
        tn = in / h;
        tm = first + in - tn * h;
    }
};

enum W8Kind : int32_t { W8_ROW = 0, W8_SPLIT = 1, W8_TILE = 2 };
// Tiles of 16 weight rows by tiles of 16 tokens of a workgroup of the tiled form
enum W8Shape : int32_t { W8_8x8 = 0, W8_14x16, W8_16x14, W8_16x16, W8_SHAPES };
constexpr int32_t kW8Sides[W8_SHAPES][2] = {{8, 8}, {14, 16}, {16, 14}, {16, 16}};
struct W8Plan {
    W8Kind kind;
    int32_t split;         // W8_ROW: wavefronts that share a tile of weights
    int32_t nt, mt;        // W8_SPLIT: tiles of a workgroup
    int32_t quant_waves;   // wavefronts that quantize a row of x: 1, 2, 4 or 8
    int32_t grid_x, grid_y;
    int64_t lds;
    W8Shape shape;         // W8_TILE
    W8Grid tiles;
};

inline W8Plan w8_plan(int32_t m, int32_t n, int32_t k, bool glu) {
    const int32_t tiles = w8_tiles(n, glu), mbs = (m + 15) / 16;
    W8Plan p{};
    if (w8_in_rows(m, k)) {
        p.kind = W8_ROW;
        const int32_t units = (n + 15) / 16;
        // Wavefronts to a tile: enough for four on each CU, and for eight where each still has 8
        // blocks (one row by 14336 x 4096: 448 workgroups 11.2 us in a graph, 224 12.7; by 32000 x
        // 2048 12.1, 13.5; but by 5632 x 2048, with 4 blocks each, 7.2, and 6.2 with 8).
        p.split = 1;
        while (p.split < kW8Waves && ((int64_t)units * p.split < 1024 ||
                                      ((int64_t)units * p.split < 2048 && w8_blocks(k) >= 16 * p.split)))
            p.split *= 2;
        const int32_t per = kW8Waves / p.split;
        p.grid_x = (units + per - 1) / per;
        p.grid_y = 1;
        p.lds = (int64_t)w8_blocks(k) * 64 * m + kW8Waves * (glu ? 2 : 1) * 1024;
        return p;
    }
    // wavefronts to a row of x, as few as hold it in registers while there are rows enough
    p.quant_waves = 8;
    while (p.quant_waves > 1 && (int64_t)m * p.quant_waves > 4096 && w8_blocks(k) * 8 <= kW8Keep * 64 * (p.quant_waves / 2))
        p.quant_waves /= 2;
    // Without LDS (tiles of nt by mt, K split over a workgroup) while 64 x 64 tiles are at most
    // 400: 128 rows by 5632 x 2048 take 11.4 us, in the tiled form 17.2, 256 rows 18.1 and 18.2,
    // 512 rows by 2048 x 5632 19.8 and 32.2; but 384 rows by 5632 x 2048 (528 tiles) 21.7 and
    // 19.7, 128 rows by 14336 x 4096 (448) 26.8 and 25.6, 48 rows of pairs of them (448) 27.5 and
    // 27.3, 100 rows (896) 50 and 30.  The rule goes by the tiles alone: up to some 32 rows of
    // still more channels the tiled form loses (8 rows of those pairs 24.3, without LDS 22.2, 32
    // rows 26.1, 23.2; by 32000 x 2048 17.6, 14.8 and 19.0, 15.8, but 64 rows 20.9, 22.0).
    auto wgs = [&](int32_t nt, int32_t mt) { return (int64_t)((tiles + nt - 1) / nt) * ((mbs + mt - 1) / mt); };
    if (wgs(4, 4) <= 400) {
        p.kind = W8_SPLIT;
        // A 4 x 4 workgroup takes as long as 3.5 of the others, and fewer than 200 no less: 32
        // rows by 14336 x 4096 take 14.6 us as 2 x 2, 20.8 as 2 x 1; 48 rows 21.5 as 2 x 2, 16.2
        // as 4 x 4; 128 rows by 2048 x 5632 12.4, 11.4, 15.8; 64 by 5632 x 2048 10.4, 9.4, 11.0.
        const int64_t one = wgs(2, 1), two = wgs(2, 2), w4 = wgs(4, 4), four = (w4 > 200 ? w4 : 200) * 7 / 2;
        p.mt = one <= two && one <= four ? 1 : two <= four ? 2 : 4;
        p.nt = p.mt == 4 ? 4 : 2;
        p.grid_x = (tiles + p.nt - 1) / p.nt;
        p.grid_y = (mbs + p.mt - 1) / p.mt;
        return p;
    }
    // The shape with the least work on the busiest CU, in units of a product of two tiles: a
    // 16 x 16 workgroup at a time on each of 256 CUs, of 8 x 8 two, which read a quarter more
    // for their products (8192^3: 450 us, 564; 1024 rows by 4096 x 4096, 64 workgroups or 256:
    // 51, 32).  One side of 14 where rounds of 256 are fuller by it: tokens' (2001 rows of 14336 x
    // 4096 pairs, 896 workgroups of 16 x 16 or 1008: 232 us, 214) or channels' (4096 rows by 14336
    // x 4096, 896 or 1024: 219 us, 212).
    p.kind = W8_TILE;
    int64_t best = INT64_MAX;
    for (int32_t i = W8_SHAPES - 1; i >= 0; i--) {
        const int32_t sn = kW8Sides[i][0], sm = kW8Sides[i][1];
        if (glu && i == W8_14x16) continue;   // a wavefront has 7 tiles of weights there: no pairs
        const int32_t at_once = i == W8_8x8 ? 512 : 256, weight = i == W8_8x8 ? 250 : i == W8_16x16 ? 100 : 106;
        const int64_t all = (int64_t)((tiles + sn - 1) / sn) * ((mbs + sm - 1) / sm);
        const int64_t cost = (all + at_once - 1) / at_once * sn * sm * weight;
        if (cost >= best) continue;
        best = cost;
        p.shape = (W8Shape)i;
        p.tiles = W8Grid{(tiles + sn - 1) / sn, (mbs + sm - 1) / sm, 8};
    }
    p.grid_x = p.tiles.n * p.tiles.m;
    p.grid_y = 1;
    return p;
}

}  // namespace tl

#if defined(__HIPCC__)

#include <hip/hip_runtime.h>

namespace tl {

enum DType : int { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2, DT_I8 = 3 };   // tl_dtype

struct PagedCache {
    PagedGeom g;
    void* k;
    void* v;
    const float* ks;   // [n_kv] (DT_I8)
    const float* vs;
    int32_t dtype;
};

struct PagedAppendArgs {
    PagedCache c;
    const void* qkv;           // [rows][(n_heads + 2 n_kv) * head_dim], stride qkv_stride
    int64_t qkv_stride;
    int32_t act;               // DType of qkv and q_out
    int32_t rows, n_heads;
    const int32_t* row_seq;    // or null: row r is sequence r
    const int32_t* row_pos;
    const float* cos;          // [n_pos][head_dim]
    const float* sin;
    int32_t n_pos;
    void* q_out;               // [rows][n_heads * head_dim], stride q_stride, or null
    int64_t q_stride;
    const float* q_gain;       // [head_dim], 16-byte aligned: q, or k, is normed first; or null
    const float* k_gain;
    double eps;
    int32_t* fault;            // set to 1 where a row names no place in the cache, or null
};
hipError_t launch_paged_append(hipStream_t s, const PagedAppendArgs& a);

// The first `len` positions of sequence `seq`, shared by all rows (len 0: none), and what
// the kernel leaves to the join: O [splits + 1][rows][n_heads][head_dim], m and l [...][2],
// and the first tile of each row's own keys [rows], then the number of all
struct PagedPrefix {
    int32_t seq, len, splits;
    float* o;
    float* ml;
    int32_t* starts;
};

struct PagedAttnArgs {
    PagedCache c;
    PagedPrefix prefix;
    const void* q;             // [rows][n_heads * head_dim], stride q_stride
    int64_t q_stride;
    int32_t act;
    int32_t rows, n_heads;
    const int32_t* row_seq;
    const int32_t* row_pos;
    float scale;
    void* out;                 // as q, stride out_stride
    int64_t out_stride;
    float* scratch;            // paged_attention_scratch() bytes
    int32_t* counters;         // kOpCounters zeros, left zero, or null: parts are joined by a second kernel
    int32_t* fault;
};
constexpr int32_t kOpCounters = 16384;
int32_t paged_attention_workgroups(const PagedCache& c, int32_t rows, int32_t n_heads);
size_t paged_attention_scratch(const PagedCache& c, int32_t rows, int32_t n_heads);
hipError_t launch_paged_attention(hipStream_t s, const PagedAttnArgs& a);
// with a shared prefix (launch_paged_attention calls it): its scratch, and the places in it
size_t paged_shared_scratch(const PagedCache& c, int32_t rows, int32_t n_heads, int32_t len);
void paged_shared_places(PagedAttnArgs& a);
hipError_t launch_shared_attention(hipStream_t s, const PagedAttnArgs& a);
hipError_t init_prefix_kernels();

// Projections with 4-bit weights.  Packed weights (launch_pack_w4) hold, for each
// 16 rows and 128 columns, 1 KiB in the order a wavefront's lanes take it, rows and
// columns behind the last ones zero, and behind all of them the scales
// [16 rows][group][row] of scale_dtype.
struct W4Args {
    const void* x;             // [m][k] of act, stride x_stride
    int64_t x_stride;
    int32_t act;
    int32_t m, n, k, group;
    const void* packed;
    int32_t scale_dtype;
    const void* residual;      // [m][n] of act, stride res_stride, or null
    int64_t res_stride;
    void* y;                   // [m][n] of act, stride y_stride
    int64_t y_stride;
    void* scratch;             // w4_scratch() bytes, 16-byte aligned
};
bool w4_supported(int32_t k, int32_t group);
int64_t w4_packed_bytes(int32_t n, int32_t k, int32_t group, int32_t scale_dtype);
hipError_t launch_linear_w4(hipStream_t s, const W4Args& a);
// q [n][k / 2] bytes: column 2 j of a row in byte j's low nibble, 2 j + 1 in its
// high one, each a two's complement number -8 .. 7; scales [n][k / group]
hipError_t launch_pack_w4(hipStream_t s, const uint8_t* q, const void* scales, int32_t scale_dtype, int32_t group,
                          int32_t n, int32_t k, void* packed);
hipError_t launch_quantize_w4(hipStream_t s, const float* w, int32_t rows, int32_t k, int32_t group, int32_t scale_dtype,
                              uint8_t* q, void* scales);
hipError_t init_w4_kernels();

// Projections with 8-bit weights (launch_pack_w8) and rows quantized on the way
struct W8Args {
    const void* x;             // [m][k] of act, stride x_stride, any alignment of the type
    int64_t x_stride;
    int32_t act;
    int32_t m, n, k;
    const void* packed;
    bool glu;                  // packed holds gate and up: y = silu(gate) up
    const void* residual;      // [m][n] of act, stride res_stride, or null
    int64_t res_stride;
    void* y;                   // [m][n] of act, stride y_stride
    int64_t y_stride;
    void* scratch;             // w8_scratch() bytes, 16-byte aligned
};
hipError_t launch_linear_w8(hipStream_t s, const W8Args& a);
// q [n][k] and scales [n]; with q2 and scales2, gate and up
hipError_t launch_pack_w8(hipStream_t s, const int8_t* q, const float* scales, const int8_t* q2, const float* scales2,
                          int32_t n, int32_t k, void* packed);

// log probabilities, entropy and top alternatives of rows of logits
struct LogprobsArgs {
    const void* logits;        // [rows][vocab] of dtype, stride `stride`, any alignment of the type
    int64_t stride;
    int32_t dtype;
    int32_t rows, vocab, top;
    const int32_t* targets;    // [rows]; negative: none
    float* logprob;            // [rows]
    float* entropy;            // [rows] or null
    int32_t* top_ids;          // [rows][top]
    float* top_logprobs;       // [rows][top]
    void* scratch;             // logprobs_scratch() bytes, 16-byte aligned
    int32_t* counters;         // as PagedAttnArgs::counters
    int32_t* fault;            // set to 1 by a target from vocab on, or null
};
constexpr int32_t kMaxTop = 32;
int64_t logprobs_workgroups(int32_t rows, int32_t vocab, int32_t top);
size_t logprobs_scratch(int32_t rows, int32_t vocab, int32_t top);
hipError_t launch_token_logprobs(hipStream_t s, const LogprobsArgs& a);

}  // namespace tl
#endif  // __HIPCC__
