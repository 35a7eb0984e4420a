// tl_serving.h -- declarations of the serving operators (paged KV cache, 4-bit
// projections, token log probabilities), shared by their kernels (tl_paged.hip,
// tl_w4.hip, tl_score.hip) and the C++ runtime (tl_runtime.hip).  The index
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
    int32_t* fault;            // set to 1 where a row names no place in the cache, or null
};
hipError_t launch_paged_append(hipStream_t s, const PagedAppendArgs& a);

struct PagedAttnArgs {
    PagedCache c;
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
