// tl_paged.hip -- the paged KV cache: append with rotation, and the attention of
// one query row per token over it.
#include <algorithm>

#include "tl_rows.h"

namespace tl {
namespace {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// append: q and k of each row rotated at its position (TL:69-80, the steps of
// tl_rope: two products and their sum, each rounded to float32), k and v written
// to the row's place in the cache (INT8: clip(rne(x / s), +-127) with a float32
// division, as tl_qkv_append), q written out in the activations' type.
// A workgroup takes 256 units of one row: a unit is four rotated pairs (d ..
// d + 3 and their partners half a head on), or eight values of v.  Nothing is
// read twice from memory; the row's cos and sin are shared by its heads through
// the cache.  What bounds it: from one row to some hundreds the chain of loads and
// the launch (3.5 us for 1 row as for 61); 2048 rows of 32 + 2 x 8 heads of 128 in
// float16, 51 MB, take 11.5 us (4.5 TB/s).  A row's values are loaded before its place is
// known, and the activations' type is the compiler's: with the type looked at per
// load, loads wait for each other, 12.7 us.
// ---------------------------------------------------------------------------
TL_DEV void cache_store4(void* base, int64_t i, int dt, v4f v, float s) {
    if (dt != DT_I8) {
        store4(base, i, dt, v);
        return;
    }
    unsigned w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) w |= (unsigned)(uint8_t)sat_i8(__builtin_rintf(__fdiv_rn(v[j], s))) << (8 * j);
    *(unsigned*)((int8_t*)base + i) = w;
}

template <int ACT>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    const PagedGeom& g = a.c.g;
    const int row = blockIdx.x;
    const int hd = g.head_dim, half = hd >> 1, quads = half >> 2;
    const int n_rot = (a.n_heads + g.n_kv) * quads;
    const int u = blockIdx.y * 256 + threadIdx.x;
    const bool rotate = u < n_rot;
    const int head = rotate ? u / quads : a.n_heads + g.n_kv, w = (u - n_rot) * 8;   // (v: the head's place from w)
    const int d = rotate ? (u - head * quads) * 4 : w;
    if (!rotate && w >= g.n_kv * hd) return;
    if (head < a.n_heads && !a.q_out) return;
    // the values, on their way while the row's place is looked up
    const int64_t at = (int64_t)row * a.qkv_stride + (int64_t)head * hd + d;
    const v4f x1 = load4(a.qkv, at, ACT), x2 = load4(a.qkv, at + (rotate ? half : 4), ACT);
    const int seq = a.row_seq ? a.row_seq[row] : row;
    const int pos = a.row_pos[row];
    const PagedRow kind = paged_row_kind(g, seq, pos);
    if (kind == PAGED_ROW_PADDING) return;
    // a position needs its rotation and, for k and v, its page
    const int page = kind == PAGED_ROW_OK && pos >= 0 && pos < a.n_pos ? paged_page(g, seq, pos) : -1;
    if (page < 0) {
        if (a.fault) *a.fault = 1;
        return;
    }
    if (rotate) {
        const float* c = a.cos + (int64_t)pos * hd + d;
        const float* s = a.sin + (int64_t)pos * hd + d;
        const v4f c1 = *(const v4f*)c, c2 = *(const v4f*)(c + half), s1 = *(const v4f*)s, s2 = *(const v4f*)(s + half);
        v4f y1, y2;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            y1[j] = x1[j] * c1[j] + -x2[j] * s1[j];
            y2[j] = x2[j] * c2[j] + x1[j] * s2[j];
        }
        if (head < a.n_heads) {
            const int64_t to = (int64_t)row * a.q_stride + (int64_t)head * hd + d;
            store4(a.q_out, to, ACT, y1);
            store4(a.q_out, to + half, ACT, y2);
        } else {
            const int kvh = head - a.n_heads;
            const float sk = a.c.dtype == DT_I8 ? a.c.ks[kvh] : 1.0f;
            const int64_t to = paged_row(g, page, kvh, pos) + d;
            cache_store4(a.c.k, to, a.c.dtype, y1, sk);
            cache_store4(a.c.k, to + half, a.c.dtype, y2, sk);
        }
        return;
    }
    const int kvh = w / hd;
    const float sv = a.c.dtype == DT_I8 ? a.c.vs[kvh] : 1.0f;
    const int64_t to = paged_row(g, page, kvh, pos) + (w - kvh * hd);
    cache_store4(a.c.v, to, a.c.dtype, x1, sv);
    cache_store4(a.c.v, to + 4, a.c.dtype, x2, sv);
}

// ---------------------------------------------------------------------------
// attention of one query row per token.
//
// out_h = sum_t p_t v_t, p = softmax_t(scale q_h . k_t), t = 0 .. pos, in one
// pass over the keys with a running maximum m and sum l (base-2 exponents).
//
// Both products run on v_mfma_f32_16x16x32 with the query heads as columns:
//   S^T = K Q^T   rows: 16 keys, columns: heads
//   O^T = V^T P^T rows: 16 dimensions, columns: heads
// A column's maximum, sum and rescaling then belong to one lane's column, and
// the probabilities a lane computes from S^T are the operand it feeds to the
// second product, with no exchange: the key rows of the two S^T tiles of 32 keys
// are chosen so that lane group g (lane / 16) holds keys 8 g .. 8 g + 7.
// The same 8 keys of V arrive as rows of consecutive dimensions (dimension
// HD/16 m + j for lane m of a group, product j) and are paired up in registers.
//
// Precision: only 8 of the 16 columns are needed (up to 8 query heads of a KV
// head per workgroup), so each head has two: one with the leading bits of q or
// p in the 16-bit type, one with the rest.  Two float16 parts, each rounded to
// nearest, are within 2^-23 of a float32 number (or, far below the row's largest,
// within 2^-38 of that); an exact 16-bit q uses the second column for nothing.  Two
// bfloat16 parts hold 16 bits: probabilities over a bfloat16 cache take a second
// product with the third part, which makes them whole, and so does q of other
// activations (X2).  INT8 keys and values are float16 integers, exactly.
//
// What bounds it: memory where the cache is long (40 ragged rows of up to 8192 keys,
// 32 / 8 heads of 128: bfloat16 120 us, 5.6 TB/s; float32 rows over bfloat16 121, over
// float16 118), else the chain of loads and the join of the parts.  The third parts
// cost 1 us of the first.
// ---------------------------------------------------------------------------
template <bool BF>
TL_DEV v4f mfma32(v4i a, v4i b, v4f c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// two INT8 values (one in each 16-bit half, zero extended) as float16: 0x6400 | u
// is 1024 + u for u < 1024, and u = x ^ 0x80 is x + 128, so 1152 less is x exactly
TL_DEV int i8_pair_f16(unsigned halves) {
    const h2 v = __builtin_bit_cast(h2, halves ^ 0x64806480u);
    return __builtin_bit_cast(int, v - h2{(_Float16)1152.0f, (_Float16)1152.0f});
}

// two floats to the 16-bit type: bfloat16 truncated, float16 to nearest
template <bool BF>
TL_DEV int pack2(float a, float b) {
    if constexpr (BF) return (int)__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    else return __builtin_bit_cast(int, h2{(_Float16)a, (_Float16)b});
}

// W dwords read once
template <int W>
TL_DEV void load_row(const char* p, unsigned v[W]) {
    typedef unsigned vec __attribute__((ext_vector_type(W)));
    if constexpr (W == 1) {
        v[0] = __builtin_nontemporal_load((const unsigned*)p);
    } else {
        const vec x = __builtin_nontemporal_load((const vec*)p);
#pragma unroll
        for (int i = 0; i < W; i++) v[i] = x[i];
    }
}

TL_DEV float pair_max(float v) {   // maximum over the four 16-lane groups
    const unsigned u = __float_as_uint(v);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float w = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const unsigned x = __float_as_uint(w);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kAttnWaves = 4;
constexpr int kAttnThreads = 64 * kAttnWaves;
constexpr int kJoinParts = 16;   // parts per (row, head block) up to which they are joined in place

template <int HD, int DT, bool X2>
struct PagedTile {
    static constexpr bool BF = DT == DT_BF16;
    static constexpr int ES = DT == DT_I8 ? 1 : 2;       // bytes per cached value
    static constexpr int KC = HD / 32;                   // S products per 16 keys
    static constexpr int ROW = HD * ES;                  // bytes of a cached row
    static constexpr int KN = 32 * ROW / 1024;           // 16-byte loads of 32 key rows per lane
    // Adjacent lanes load adjacent 16-byte pieces of one row, up to 128 bytes of it;
    // the products want a row's pieces 16 lanes apart, so they pass through LDS.
    static constexpr int KC_LINE = ROW < 128 ? ROW / 16 : 8;   // pieces of a row in one load
    static constexpr int KR = 64 / KC_LINE;              // rows in one load
    static constexpr int KLINES = ROW / (16 * KC_LINE);  // loads of a row
    // piece `piece` of a row m of 16 stands at slot piece ^ swizzle(m): eight
    // lanes reading one piece of their rows then meet 32 different banks twice
    TL_DEV static int swizzle(int m) { return KC_LINE == 8 ? m & 7 : m >> 2 & 3; }
    // where 16-byte unit u of row m of tile t stands
    TL_DEV static int slot(int t, int m, int u) {
        const int r = t * 16 + m;
        return ((r / KR * KLINES + u / KC_LINE) * 64 + r % KR * KC_LINE + (u % KC_LINE ^ swizzle(m))) * 16;
    }
    static constexpr int LDS = 32 * ROW > 8 * (HD + 4) * 4 ? 32 * ROW : 8 * (HD + 4) * 4;   // a wavefront's bytes
    static constexpr int VD = HD / 16;                   // dimensions of V per lane: O products
    static constexpr int VW = VD * ES / 4;               // dwords of a V row per lane
    static constexpr int QP = X2 ? 2 : 1;                // products of q's parts
    static constexpr int PP = BF ? 2 : 1;                // and of the probabilities'

    // first dimension of the 8 that lane group g multiplies in S product c
    TL_DEV static int q_dim(int c, int g) { return DT == DT_I8 ? (c >> 1) * 64 + 16 * g + 8 * (c & 1) : (c * 4 + g) * 8; }
};

// A part's numbers in scratch: O of 8 heads [8][HD], then m and l of each
template <int HD>
TL_DEV float* part_o(const PagedAttnArgs& a, int32_t part) { return a.scratch + (int64_t)part * 8 * HD; }
template <int HD>
TL_DEV float* part_ml(const PagedAttnArgs& a, int32_t part, int32_t workgroups) {
    return a.scratch + (int64_t)2 * workgroups * 8 * HD + (int64_t)part * 16;
}

// this thread's row of the rows scanned together (kAttnThreads at a time), its tiles
TL_DEV unsigned row_tiles(const PagedAttnArgs& a, int64_t row) {
    if (row >= a.rows) return 0u;
    const int seq = a.row_seq ? a.row_seq[row] : (int)row;
    const int pos = a.row_pos[row];
    return paged_row_kind(a.c.g, seq, pos) == PAGED_ROW_OK ? (unsigned)paged_tiles(pos + 1) : 0u;
}

struct ScanShared {
    unsigned wave[kAttnWaves];
    int32_t before, row;
};

// inclusive sums over the workgroup's threads; all: the sum
TL_DEV unsigned block_scan(unsigned v, ScanShared& sh, unsigned& all) {
    const int lane = lane_id(), wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned up = (unsigned)__shfl_up((int)v, o);
        if (lane >= o) v += up;
    }
    __syncthreads();
    if (lane == 63) sh.wave[wave] = v;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < kAttnWaves; w++) {
        if (w < wave) v += sh.wave[w];
        all += sh.wave[w];
    }
    return v;
}

// tiles of the rows scanned together: this thread's row's, the sum up to it, and all
struct RowScan {
    unsigned mine, upto, all;
};
TL_DEV RowScan scan_rows(const PagedAttnArgs& a, ScanShared& sh, int64_t r0) {
    RowScan r;
    r.mine = row_tiles(a, r0 + threadIdx.x);
    r.upto = block_scan(r.mine, sh, r.all);
    return r;
}

// The call's rows in a wavefront's lanes (up to 64 rows): no barrier, and a row's
// sequence and position at hand for the whole kernel.
struct LaneRows {
    int seq, pos;
    unsigned tiles, upto;
};
TL_DEV LaneRows lane_rows(const PagedAttnArgs& a, unsigned& all) {
    const int r = min(lane_id(), a.rows - 1);
    LaneRows l;
    l.seq = a.row_seq ? a.row_seq[r] : r;
    l.pos = a.row_pos[r];
    const bool use = lane_id() < a.rows && paged_row_kind(a.c.g, l.seq, l.pos) == PAGED_ROW_OK;
    l.tiles = use ? (unsigned)paged_tiles(l.pos + 1) : 0u;
    unsigned v = l.tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned up = (unsigned)__shfl_up((int)v, o);
        if (lane_id() >= o) v += up;
    }
    l.upto = v;
    all = (unsigned)__builtin_amdgcn_readlane((int)v, 63);
    return l;
}

// the call's tiles per head block; first: the first scan's
TL_DEV int32_t count_tiles(const PagedAttnArgs& a, ScanShared& sh, RowScan& first) {
    first = scan_rows(a, sh, 0);
    int32_t total = (int32_t)first.all;
    for (int64_t r0 = kAttnThreads; r0 < a.rows; r0 += kAttnThreads) {
        unsigned all;
        block_scan(row_tiles(a, r0 + threadIdx.x), sh, all);
        total += (int32_t)all;
    }
    return total;
}

// the row that holds tile `at` (of one head block, at < total) and the tiles before that row
TL_DEV void find_row(const PagedAttnArgs& a, ScanShared& sh, int32_t at, RowScan r, int& row, int32_t& before) {
    int32_t base = 0;
    for (int64_t r0 = 0;;) {
        const int32_t end = base + (int32_t)r.upto, start = end - (int32_t)r.mine;
        if (start <= at && at < end) {
            sh.before = start;
            sh.row = (int32_t)(r0 + threadIdx.x);
        }
        base += (int32_t)r.all;
        r0 += kAttnThreads;
        if (at < base || r0 >= a.rows) break;
        r = scan_rows(a, sh, r0);
    }
    __syncthreads();
    row = __builtin_amdgcn_readfirstlane(sh.row);
    before = __builtin_amdgcn_readfirstlane(sh.before);
}

// Parts that another workgroup joins go through to memory as they are written and
// are read from there: loads and stores of agent scope.  The other way, plain
// stores and a release fence, writes the whole L2 back: with 512 workgroups
// leaving parts it took the kernel from 13 to 45 us (32 rows of 1984 keys).
TL_DEV void part_store4(float* p, v4f v) {
    typedef unsigned long long u64;
    const v2f lo = {v[0], v[1]}, hi = {v[2], v[3]};
    __hip_atomic_store((u64*)p, __builtin_bit_cast(u64, lo), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store((u64*)p + 1, __builtin_bit_cast(u64, hi), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
TL_DEV v2f part_load2(const float* p) {
    return __builtin_bit_cast(v2f, __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
TL_DEV v4f part_load4(const float* p) {
    const v2f lo = part_load2(p), hi = part_load2(p + 2);
    return v4f{lo[0], lo[1], hi[0], hi[1]};
}

// The parts w0 .. w1 of a (row, head block) joined by one workgroup, in the order of
// their keys: M = max m, out = sum 2^(m - M) O / sum 2^(m - M) l, kJoinStep parts
// at a time.
constexpr int kJoinStep = 32;
struct JoinShared {
    float e[kJoinStep][8], l[kJoinStep][8];   // 2^(m - M) (first m) and l of each part
    float m[8], sum[8], keep[8];              // M and the sum so far, what the parts before are scaled by
};
template <int HD>
TL_DEV void join_parts(const PagedAttnArgs& a, const PagedShare& share, int w0, int w1, int32_t unit, int row,
                       int64_t head0, int heads, JoinShared& sh) {
    const int h = threadIdx.x / (HD / 4), d = (threadIdx.x - h * (HD / 4)) * 4;   // this thread's four values
    v4f acc = {0, 0, 0, 0};
    for (int p0 = w0; p0 <= w1; p0 += kJoinStep) {
        const int parts = min(kJoinStep, w1 - p0 + 1);
        if ((int)threadIdx.x < parts * 8) {
            const int p = threadIdx.x >> 3, k = threadIdx.x & 7;
            const v2f ml = part_load2(part_ml<HD>(a, paged_part(share, p0 + p, unit), gridDim.x) + 2 * k);
            sh.e[p][k] = ml[0];
            sh.l[p][k] = ml[1];
        }
        v4f v[8];
        auto load8 = [&](int at) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                v[j] = part_load4(part_o<HD>(a, paged_part(share, min(p0 + at + j, w1), unit)) + h * HD + d);
        };
        if (h < heads) load8(0);
        __syncthreads();
        if (threadIdx.x < 8) {
            const int k = threadIdx.x;
            const float before = p0 == w0 ? -__builtin_inff() : sh.m[k];
            float mm = before;
            for (int p = 0; p < parts; p++) mm = fmaxf(mm, sh.e[p][k]);
            const float off = mm == -__builtin_inff() ? 0.0f : mm;
            const float keep = __builtin_amdgcn_exp2f(before - off);
            float ll = p0 == w0 ? 0.0f : sh.sum[k] * keep;
            for (int p = 0; p < parts; p++) {
                const float e = __builtin_amdgcn_exp2f(sh.e[p][k] - off);
                ll += e * sh.l[p][k];
                sh.e[p][k] = e;
            }
            sh.m[k] = mm;
            sh.sum[k] = ll;
            sh.keep[k] = keep;
        }
        __syncthreads();
        if (h < heads) {
            acc *= sh.keep[h];
            for (int at = 0; at < parts; at += 8) {   // eight parts' loads at once
                if (at > 0) load8(at);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (at + j < parts) acc += sh.e[at + j][h] * v[j];
            }
        }
        __syncthreads();
    }
    if (h < heads) store4(a.out, (int64_t)row * a.out_stride + (head0 + h) * HD + d, a.act, acc / sh.sum[h]);
}

// The pages of the four groups of 8 keys of 32, each in one page; groups behind the
// last key are looked up where it is.  Bit j of bad: group j's page is out of range
// (page 0 is read in its place and does not count).  The table is read by scalar
// loads: their counter is not the rows', which stay in flight.
struct PagedPlace {
    unsigned p0, p1, p2, p3;
    unsigned bad;
};
typedef const __attribute__((address_space(4))) int32_t* scalar_table;
// group i's page: by selects of masks, as an indexed choice among the fields puts the
// struct into memory (LDS, and its address costs a read of the launch's packet)
TL_DEV unsigned pick_page(PagedPlace p, int i) {
    const unsigned odd = 0u - (unsigned)(i & 1), high = 0u - (unsigned)(i >> 1 & 1);
    const unsigned a = p.p0 ^ ((p.p0 ^ p.p1) & odd), b = p.p2 ^ ((p.p2 ^ p.p3) & odd);
    return a ^ ((a ^ b) & high);
}

TL_DEV PagedPlace place_rows(const PagedGeom& geo, scalar_table row, int kb, int last8) {
    PagedPlace p;
    p.bad = 0;
    auto look = [&](int j) {
        const unsigned page = (unsigned)row[min(kb + 8 * j, last8) >> geo.page_shift];
        const bool in = page < (unsigned)geo.n_pages;
        p.bad |= in ? 0u : 1u << j;
        return in ? page : 0u;
    };
    p.p0 = look(0);
    if (geo.page_shift >= 5) {   // 32 keys from a multiple of 32 on: one page
        p.p1 = p.p2 = p.p3 = p.p0;
        p.bad = p.bad ? 15u : 0u;
    } else {
        p.p1 = look(1);
        p.p2 = look(2);
        p.p3 = look(3);
    }
    return p;
}

// where a lane's group of 8 keys starts: a page and 32 bits of bytes in it
template <int BYTES>   // of a row
TL_DEV const char* group_row(const char* base, const PagedGeom& geo, unsigned page_bytes, unsigned page, int key) {
    const unsigned at = (unsigned)(key & ((1 << geo.page_shift) - 1)) * BYTES;
    return base + ((uint64_t)page * page_bytes + at);
}

// Key rows of S^T: row m of tile t is key 8 (m / 4) + 4 t + m % 4 of the 32
template <int HD, int DT, bool X2>
TL_DEV void load_keys(const PagedGeom& geo, const char* base, unsigned page_bytes, int kb, int last8, int lane,
                      PagedPlace p, v4i kf[PagedTile<HD, DT, X2>::KN]) {
    using T = PagedTile<HD, DT, X2>;
#pragma unroll
    for (int rb = 0; rb < 32 / T::KR; rb++) {
        const int r = rb * T::KR + lane / T::KC_LINE, m = r & 15, t = r >> 4, grp = m >> 2;
        const char* kr = group_row<T::ROW>(base, geo, page_bytes, pick_page(p, grp), min(kb + 8 * grp, last8)) +
                         (4 * t + (m & 3)) * T::ROW + 16 * (lane % T::KC_LINE);
#pragma unroll
        for (int i = 0; i < T::KLINES; i++)
            kf[rb * T::KLINES + i] = __builtin_nontemporal_load((const v4i*)(kr + i * 16 * T::KC_LINE));
    }
}

template <int HD, int DT, bool X2>
TL_DEV void load_values(const PagedGeom& geo, const char* base, unsigned page_bytes, int kb, int last8, int col, int g,
                        PagedPlace p, unsigned vf[8][PagedTile<HD, DT, X2>::VW]) {
    using T = PagedTile<HD, DT, X2>;
    const char* vr = group_row<HD * T::ES>(base, geo, page_bytes, pick_page(p, g), min(kb + 8 * g, last8)) + col * (T::VW * 4);
#pragma unroll
    for (int j = 0; j < 8; j++) load_row<T::VW>(vr + j * HD * T::ES, vf[j]);
}

// A workgroup works through its run of tiles: the end of one (row, head block),
// whole ones, the start of another.  Of each, its wavefronts take every fourth
// 32 keys with their own m, l and O, joined through LDS; a whole one is finished,
// of the others a part is left in scratch.  With counters the workgroup that
// leaves the last part of a (row, head block) joins them, else a second kernel.
template <int HD, int DT, bool X2>
__global__ __launch_bounds__(kAttnThreads, 2) void paged_attention_kernel(PagedAttnArgs a) {
    using T = PagedTile<HD, DT, X2>;
    constexpr bool BF = T::BF;
    __shared__ __align__(16) char s_wave[kAttnWaves][T::LDS];   // key rows on their way, then O [8][HD + 4]
    __shared__ float s_m[kAttnWaves][8], s_l[kAttnWaves][8];
    __shared__ ScanShared s_scan;
    __shared__ JoinShared s_join;
    __shared__ int s_last;
    const PagedGeom& geo = a.c.g;
    const int rep = a.n_heads / geo.n_kv;
    const int blocks = (rep + 7) >> 3, hbs = geo.n_kv * blocks;
    const int lane = lane_id(), wave = wave_id(), col = lane & 15, g = lane >> 4;
    const bool lo = col >= 8;
    const int head = col & 7;
    char* const my_lds = s_wave[wave];
    // where this lane's pieces go (its rows of 16 are alike in swizzle whatever the load)
    const int key_slot = (lane ^ T::swizzle(lane / T::KC_LINE)) * 16;
    const int me = blockIdx.x;

    const bool few = a.rows <= kPagedFewRows;
    RowScan first = {};
    LaneRows lr = {};
    int32_t total;
    if (few) {
        unsigned all;
        lr = lane_rows(a, all);
        total = (int32_t)all;
    } else {
        total = count_tiles(a, s_scan, first);
    }
    if (me == 0 && a.fault)
        for (int64_t r = threadIdx.x; r < a.rows; r += kAttnThreads)
            if (paged_row_kind(geo, a.row_seq ? a.row_seq[r] : (int)r, a.row_pos[r]) == PAGED_ROW_FAULT) *a.fault = 1;
    const PagedShare share = paged_share(__builtin_amdgcn_readfirstlane(total) * hbs, gridDim.x);
    int32_t at = share.start(me);
    const int32_t stop = share.start(me + 1);
    if (at >= stop) return;
    int row;
    int32_t before;
    if (few) {
        const unsigned tile = (unsigned)at / (unsigned)hbs;
        row = __builtin_ctzll(__builtin_amdgcn_ballot_w64(tile < lr.upto));
        before = __builtin_amdgcn_readlane((int)(lr.upto - lr.tiles), row);
    } else {
        find_row(a, s_scan, (unsigned)at / (unsigned)hbs, first, row, before);
    }
    // tile `at` of all lies `in` tiles into its row's head blocks
    int32_t in = at - before * hbs;
    bool bad = false;

    for (; at < stop; row++) {
        const int seq = few ? __builtin_amdgcn_readlane(lr.seq, row) : a.row_seq ? a.row_seq[row] : row;
        const int pos = few ? __builtin_amdgcn_readlane(lr.pos, row) : a.row_pos[row];
        if (paged_row_kind(geo, seq, pos) != PAGED_ROW_OK) continue;
        const int n = __builtin_amdgcn_readfirstlane(max(pos + 1, 0));
        const int tiles = paged_tiles(n);
        for (int hb = (int)((unsigned)in / (unsigned)tiles); hb < hbs && at < stop; hb++) {
            const int t0 = in - hb * tiles;
            const int t1 = min(tiles, t0 + (stop - at));
            const int32_t unit = at - t0;   // the (row, head block)'s first tile
            at += t1 - t0;
            in = (hb + 1) * tiles;
            const int kvh = hb / blocks, h0 = (hb - kvh * blocks) * 8;
            const int heads = min(8, rep - h0);
            const int64_t head0 = (int64_t)kvh * rep + h0;
            if (n == 0) {   // no keys: zeros
                for (int i = threadIdx.x; i < heads * HD / 4; i += kAttnThreads)
                    store4(a.out, (int64_t)row * a.out_stride + head0 * HD + 4 * i, a.act, v4f{0, 0, 0, 0});
                continue;
            }
            const int end = min(n, t1 * kPagedTile);
            const int last8 = (n - 1) & ~7;
            int kb = t0 * kPagedTile + 32 * wave;
            const scalar_table table = (scalar_table)(geo.table + (int64_t)seq * geo.table_stride);
            const unsigned page_bytes = (unsigned)(geo.page_stride * T::ES);
            const unsigned head_bytes = ((unsigned)kvh << geo.page_shift) * (HD * T::ES);
            const char* kbase = (const char*)a.c.k + head_bytes;
            const char* vbase = (const char*)a.c.v + head_bytes;
            // a lane's pieces of the key rows and 8 rows of V, of 32 keys
            v4i kf[T::KN];
            unsigned vf[8][T::VW];
            unsigned pages_bad = 0;
            auto fetch = [&](int key) {
                const PagedPlace place = place_rows(geo, table, key, last8);
                pages_bad = place.bad;
                load_keys<HD, DT, X2>(geo, kbase, page_bytes, key, last8, lane, place, kf);
                load_values<HD, DT, X2>(geo, vbase, page_bytes, key, last8, col, g, place, vf);
            };
            fetch(kb);   // (a wavefront without keys: the last ones)
            // the query head's parts, scaled by a power of two so that float16 holds them
            v4i qf[T::QP][T::KC];
            float cs = a.scale * kLog2e;
            if constexpr (DT == DT_I8) cs *= a.c.ks[kvh];
            {
                float q[T::KC][8];
                float mx = 0.0f;
                const int64_t qat = (int64_t)row * a.q_stride + (head0 + min(head, heads - 1)) * HD;
#pragma unroll
                for (int c = 0; c < T::KC; c++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const v4f v = load4(a.q, qat + T::q_dim(c, g) + 4 * h, a.act);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            q[c][4 * h + j] = v[j];
                            mx = fmaxf(mx, fabsf(v[j]));
                        }
                    }
                }
                float up = 1.0f;
                if constexpr (!BF) {
                    mx = pair_max(mx);
                    // max |q| in [2^13, 2^14): an infinite, NaN or zero row stays as it is
                    const int e = mx > 0.0f && mx < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(mx) : 0;
                    up = __builtin_amdgcn_ldexpf(1.0f, min(e, 126));
                    cs = __builtin_amdgcn_ldexpf(cs, -min(e, 126));
                }
#pragma unroll
                for (int c = 0; c < T::KC; c++) {
                    float part[T::QP][8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float x = q[c][j] * up;
                        float hi, mid;
                        if constexpr (BF) {
                            hi = (float)(__bf16)x;
                            mid = (float)(__bf16)(x - hi);
                        } else {
                            hi = (float)(_Float16)x;
                            mid = x - hi;
                        }
                        part[0][j] = lo ? mid : hi;
                        if constexpr (X2) part[1][j] = lo ? 0.0f : x - hi - mid;
                    }
#pragma unroll
                    for (int p = 0; p < T::QP; p++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float x = part[p][2 * j], y = part[p][2 * j + 1];
                            qf[p][c][j] = (int)(BF ? to_bf16(x) | (to_bf16(y) << 16) : to_f16(x) | (to_f16(y) << 16));
                        }
                }
            }

            float m = -__builtin_inff(), l = 0.0f;
            v4f o[T::VD];
#pragma unroll
            for (int j = 0; j < T::VD; j++) o[j] = v4f{0, 0, 0, 0};
            const unsigned lo_mask = lo ? 0xFFFFFFFFu : 0u;

            while (kb < end) {
#pragma unroll
                for (int j = 0; j < T::KN; j++) *(v4i*)(my_lds + j * 1024 + key_slot) = kf[j];
                __builtin_amdgcn_wave_barrier();
                v4f s[2] = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}};
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int c = 0; c < T::KC; c++) {
                        v4i kk;
                        if constexpr (DT == DT_I8) {
                            const v2i w = *(const v2i*)(my_lds + T::slot(t, col, (c >> 1) * 4 + g) + 8 * (c & 1));
                            const unsigned w0 = (unsigned)w[0], w1 = (unsigned)w[1];
                            kk = v4i{i8_pair_f16(__builtin_amdgcn_perm(0u, w0, 0x0C010C00u)), i8_pair_f16(__builtin_amdgcn_perm(0u, w0, 0x0C030C02u)),
                                     i8_pair_f16(__builtin_amdgcn_perm(0u, w1, 0x0C010C00u)), i8_pair_f16(__builtin_amdgcn_perm(0u, w1, 0x0C030C02u))};
                        } else {
                            kk = *(const v4i*)(my_lds + T::slot(t, col, c * 4 + g));
                        }
#pragma unroll
                        for (int p = 0; p < T::QP; p++) s[t] = mfma32<BF>(kk, qf[p][c], s[t]);
                    }
                __builtin_amdgcn_wave_barrier();

                // lane: keys kb + 8 g + 4 t + i of its head, both parts' products added
                float x[8], mt = -__builtin_inff();
                const bool whole = kb + 32 <= n && pages_bad == 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float d = s[j >> 2][j & 3];
                    x[j] = (d + lane_xor<8>(d)) * cs;
                }
                if (!whole) {
                    bad |= pages_bad != 0;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const bool in = !(pages_bad >> g & 1) && kb + 8 * g + j < n;
                        x[j] = in ? x[j] : -__builtin_inff();
#pragma unroll
                        for (int w = 0; w < T::VW; w++) vf[j][w] = in ? vf[j][w] : 0u;   // 0 x NaN of a stale row is NaN
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; j++) mt = fmaxf(mt, x[j]);
                mt = pair_max(mt);
                if (__builtin_amdgcn_ballot_w64(mt > m) != 0) {
                    const float mn = fmaxf(m, mt);
                    const float al = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    l *= al;
#pragma unroll
                    for (int j = 0; j < T::VD; j++) o[j] *= al;
                }
                // p 2^14, so that the float16 parts of small probabilities stay normal
                const float off = m == -__builtin_inff() ? 0.0f : (BF ? m : m - 14.0f);
                v4i pf[T::PP];
                {
                    float part[T::PP][8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float p = __builtin_amdgcn_exp2f(x[j] - off);
                        l += p;
                        // the leading part (the pack rounds it off), or what it leaves
                        const float hi = BF ? __uint_as_float(__float_as_uint(p) & 0xFFFF0000u) : (float)(_Float16)p;
                        part[0][j] = p - __uint_as_float(__float_as_uint(hi) & lo_mask);
                        if constexpr (BF) {
                            const float rest = p - hi;
                            part[1][j] = lo ? 0.0f : rest - __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
                        }
                    }
#pragma unroll
                    for (int p = 0; p < T::PP; p++)
#pragma unroll
                        for (int j = 0; j < 4; j++) pf[p][j] = pack2<BF>(part[p][2 * j], part[p][2 * j + 1]);
                }
#pragma unroll
                for (int d = 0; d < T::VD; d++) {
                    v4i vv;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if constexpr (DT == DT_I8)
                            vv[r] = i8_pair_f16(__builtin_amdgcn_perm(vf[2 * r + 1][d >> 2], vf[2 * r][d >> 2],
                                                                      0x0C040C00u + 0x00010001u * (unsigned)(d & 3)));
                        else
                            vv[r] = (int)__builtin_amdgcn_perm(vf[2 * r + 1][d >> 1], vf[2 * r][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
                    }
#pragma unroll
                    for (int p = 0; p < T::PP; p++) o[d] = mfma32<BF>(vv, pf[p], o[d]);
                }
                // the registers' next rows
                kb += kPagedTile;
                if (kb >= end) break;
                fetch(kb);
            }
            // both parts of a head, then the wavefronts; lane: dimensions HD/4 g + VD i + d
            l += lane_xor<16>(l);
            l += lane_xor<32>(l);
#pragma unroll
            for (int d = 0; d < T::VD; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = o[d][i] + lane_xor<8>(o[d][i]);
                    if (!lo) ((float*)my_lds)[head * (HD + 4) + HD / 4 * g + T::VD * i + d] = v;
                }
            if (lane < 8) {
                s_m[wave][lane] = m;
                s_l[wave][lane] = l;
            }
            __syncthreads();
            const bool all = t0 == 0 && t1 == tiles;
            const int part = paged_part(share, me, unit);
            const float sv = DT == DT_I8 ? a.c.vs[kvh] : 1.0f;
            for (int i = threadIdx.x; i < heads * HD / 4; i += kAttnThreads) {
                const int h = i / (HD / 4), d = (i - h * (HD / 4)) * 4;
                float mm = s_m[0][h];
#pragma unroll
                for (int w = 1; w < kAttnWaves; w++) mm = fmaxf(mm, s_m[w][h]);
                const float off = mm == -__builtin_inff() ? 0.0f : mm;
                float ll = 0.0f;
                v4f acc = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < kAttnWaves; w++) {
                    const float e = __builtin_amdgcn_exp2f(s_m[w][h] - off);
                    ll += e * s_l[w][h];
                    acc += e * *(const v4f*)(s_wave[w] + (h * (HD + 4) + d) * 4);
                }
                acc *= sv;
                if (all) {
                    store4(a.out, (int64_t)row * a.out_stride + (head0 + h) * HD + d, a.act, acc / ll);
                } else {
                    part_store4(part_o<HD>(a, part) + h * HD + d, acc);
                    if (d == 0)
                        __hip_atomic_store((unsigned long long*)(part_ml<HD>(a, part, gridDim.x) + 2 * h),
                                           __builtin_bit_cast(unsigned long long, v2f{mm, ll}), __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
                }
            }
            if (!all && a.counters) {
                const int w0 = share.owner(unit), w1 = share.owner(unit + tiles - 1);
                // every wavefront's stores have arrived before the part is counted
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (threadIdx.x == 0) {
                    int* ctr = a.counters + row * hbs + hb;
                    const int got = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    s_last = got == w1 - w0;
                    if (s_last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                if (s_last) {
                    join_parts<HD>(a, share, w0, w1, unit, row, head0, heads, s_join);
                }
            }
            __syncthreads();
        }
        in = 0;
    }
    if (a.fault && bad) *a.fault = 1;
}

// the parts of one (row, head) joined, W of them side by side (paged_join_grid)
template <int HD>
__global__ __launch_bounds__(kAttnThreads) void paged_join_kernel(PagedAttnArgs a, int workgroups) {
    constexpr int Q = HD / 4, W = kAttnThreads / Q;   // quads of a row; parts taken side by side
    __shared__ float s_acc[W][HD];
    __shared__ float s_l[W], s_m[kAttnWaves];
    __shared__ ScanShared s_scan;
    const PagedGeom& geo = a.c.g;
    const int rep = a.n_heads / geo.n_kv, blocks = (rep + 7) >> 3, hbs = geo.n_kv * blocks;
    int row, head, tiles;
    int32_t unit;
    PagedShare share;
    if (a.rows <= kPagedFewRows) {
        row = blockIdx.x;
        head = blockIdx.y;
        const int pos = a.row_pos[row];
        if (paged_row_kind(geo, a.row_seq ? a.row_seq[row] : row, pos) != PAGED_ROW_OK || pos < 0) return;
        unsigned all;
        const LaneRows l = lane_rows(a, all);
        share = paged_share((int32_t)all * hbs, workgroups);
        tiles = paged_tiles(pos + 1);
        const int kvh = head / rep, hb = kvh * blocks + ((head - kvh * rep) >> 3);
        unit = __builtin_amdgcn_readlane((int)(l.upto - l.tiles), row) * hbs + hb * tiles;
    } else {
        const int w = blockIdx.x + 1;
        RowScan first;
        const int32_t total = __builtin_amdgcn_readfirstlane(count_tiles(a, s_scan, first));
        share = paged_share(total * hbs, workgroups);
        const int32_t at = share.start(w);
        if (at >= total * hbs || at == share.start(w - 1)) return;
        int32_t before;
        find_row(a, s_scan, (unsigned)at / (unsigned)hbs, first, row, before);
        tiles = paged_tiles(a.row_pos[row] + 1);
        const int32_t in = at - before * hbs;
        const int hb = (int)((unsigned)in / (unsigned)tiles), kvh = hb / blocks, h = (hb - kvh * blocks) * 8 + (int)blockIdx.y;
        unit = before * hbs + hb * tiles;
        if (h >= rep || !paged_joins_at(share, w, unit)) return;
        head = kvh * rep + h;
    }
    const int h = head % rep;
    const int w0 = share.owner(unit), w1 = share.owner(unit + tiles - 1);
    if (w0 == w1) return;   // one workgroup had all of it
    const int ml_at = 2 * (h & 7);
    float mm = -__builtin_inff();
    for (int w = w0 + threadIdx.x; w <= w1; w += kAttnThreads) mm = fmaxf(mm, part_ml<HD>(a, paged_part(share, w, unit), workgroups)[ml_at]);
    mm = wave_max_f32(mm);
    if (lane_id() == 0) s_m[threadIdx.x >> 6] = mm;
    __syncthreads();
    mm = s_m[0];
#pragma unroll
    for (int w = 1; w < kAttnWaves; w++) mm = fmaxf(mm, s_m[w]);
    const float off = mm == -__builtin_inff() ? 0.0f : mm;
    const int q = threadIdx.x % Q, s = threadIdx.x / Q;
    v4f acc = {0, 0, 0, 0};
    float ll = 0.0f;
#pragma unroll 4
    for (int w = w0 + s; w <= w1; w += W) {
        const int part = paged_part(share, w, unit);
        const float* ml = part_ml<HD>(a, part, workgroups) + ml_at;
        const float e = __builtin_amdgcn_exp2f(ml[0] - off);
        ll += e * ml[1];
        acc += e * *(const v4f*)(part_o<HD>(a, part) + (h & 7) * HD + 4 * q);
    }
    *(v4f*)&s_acc[s][4 * q] = acc;
    if (q == 0) s_l[s] = ll;
    __syncthreads();
    if (s != 0) return;
    for (int i = 1; i < W; i++) {
        acc += *(const v4f*)&s_acc[i][4 * q];
        ll += s_l[i];
    }
    store4(a.out, (int64_t)row * a.out_stride + (int64_t)head * HD + 4 * q, a.act, acc / ll);
}

int32_t head_blocks(int32_t n_heads, int32_t n_kv) { return (n_heads / n_kv + 7) / 8; }

}  // namespace

hipError_t launch_paged_append(hipStream_t s, const PagedAppendArgs& a) {
    if (a.rows <= 0) return hipSuccess;
    const int units = (a.n_heads + a.c.g.n_kv) * (a.c.g.head_dim / 8) + a.c.g.n_kv * a.c.g.head_dim / 8;
    const dim3 grid(a.rows, (units + 255) / 256), block(256);
    if (a.act == DT_F32) TL_KLAUNCH((paged_append_kernel<DT_F32>), grid, block, 0, s, a);
    else if (a.act == DT_BF16) TL_KLAUNCH((paged_append_kernel<DT_BF16>), grid, block, 0, s, a);
    else TL_KLAUNCH((paged_append_kernel<DT_F16>), grid, block, 0, s, a);
    return hipGetLastError();
}

// Workgroups of a call, no more than there can be tiles: two on each of 256 CUs, so
// that one works while the other changes rows (40 ragged rows of up to 8192 keys, 8
// KV heads: 120 us against 133 with one on each; 32 INT8 rows of 1984, 4 KV heads of
// 64: 15.6, 17.1); one where at most 64 (row, head block)s are split into long runs (8
// rows of 16384: 90.0 us against 91.5; one row of 131072, 4 KV heads: 51.1, 53.4).
int32_t paged_attention_workgroups(const PagedCache& c, int32_t rows, int32_t n_heads) {
    const int64_t units = (int64_t)rows * c.g.n_kv * head_blocks(n_heads, c.g.n_kv);
    const int64_t cap = (((int64_t)c.g.max_pages << c.g.page_shift) + kPagedTile - 1) / kPagedTile;
    return (int32_t)std::max<int64_t>(1, std::min<int64_t>(units <= 64 ? 256 : 512, units * cap));
}

size_t paged_attention_scratch(const PagedCache& c, int32_t rows, int32_t n_heads) {
    return (size_t)paged_attention_workgroups(c, rows, n_heads) * 2 * 8 * (c.g.head_dim + 2) * sizeof(float);
}

hipError_t launch_paged_attention(hipStream_t s, const PagedAttnArgs& args) {
    if (args.rows <= 0) return hipSuccess;
    PagedAttnArgs a = args;
    const int wgs = paged_attention_workgroups(a.c, a.rows, a.n_heads);
    const int64_t units = (int64_t)a.rows * a.c.g.n_kv * head_blocks(a.n_heads, a.c.g.n_kv);
    // parts of a (row, head block) are joined by the workgroup that leaves the last
    // one where there are few, else by a kernel of more workgroups
    if (units > kOpCounters || wgs > kJoinParts * units) a.counters = nullptr;
    const bool one_tile = ((int64_t)a.c.g.max_pages << a.c.g.page_shift) <= kPagedTile;   // nothing is split
    if (one_tile) a.counters = nullptr;
    const dim3 grid(wgs), block(kAttnThreads);
    const PagedJoinGrid join = paged_join_grid(a.rows, a.n_heads, a.c.g.n_kv, wgs);
    const bool x2 = a.c.dtype == DT_BF16 && a.act != DT_BF16;
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (a.c.dtype == DT_I8) TL_KLAUNCH((paged_attention_kernel<HD, DT_I8, false>), grid, block, 0, s, a);
        else if (a.c.dtype == DT_F16) TL_KLAUNCH((paged_attention_kernel<HD, DT_F16, false>), grid, block, 0, s, a);
        else if (x2) TL_KLAUNCH((paged_attention_kernel<HD, DT_BF16, true>), grid, block, 0, s, a);
        else TL_KLAUNCH((paged_attention_kernel<HD, DT_BF16, false>), grid, block, 0, s, a);
        if (!a.counters && !one_tile) TL_KLAUNCH((paged_join_kernel<HD>), dim3(join.x, join.y), block, 0, s, a, wgs);
    };
    if (a.c.g.head_dim == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
    return hipGetLastError();
}

}  // namespace tl
