// tl_prefix.hip -- attention of many rows over the keys that all of them share.
#include <algorithm>

#include "tl_attn.h"

namespace tl {
namespace {

// ---------------------------------------------------------------------------
// The query heads of all rows that read one KV head are the columns of one product: column
// c is head c % rep of row c / rep.  As in the attention of single tokens
//   S^T = K Q^T   rows: keys, columns: query heads
//   O^T = V^T P^T rows: dimensions, columns: query heads
// run on v_mfma_f32_16x16x32 with the keys of an S^T tile chosen so that a lane's
// probabilities are the operand it feeds to the second product, a running maximum and sum
// to each column.  A wavefront has 32 columns.  QW = 4: a workgroup's wavefronts have 128
// columns and share tiles of 64 keys; QW = 1: they have the same 32 columns and each its own
// tiles of 32 keys, joined at the end.  A tile's keys and values are read from their pages
// once, turned to 16 bits and, the values, on their side, and lie in LDS in the order of
// the products' operands.
//
// The keys are split over workgroups; each leaves O, m and l of its columns in scratch.  In
// the same launch other workgroups take the rows' own keys as paged_attention_kernel does
// (attention_run); a second kernel joins what both left.
//
// Precision: q enters in QP 16-bit parts and the probabilities in PP, as many as it takes:
// of 16-bit rows q is exact in one (float16 holds a bfloat16 scaled to its row); float32 rows
// take two float16 parts (within 2^-23) or three bfloat16 ones (whole).  Probabilities of 16-bit rows take
// two parts, as one bfloat16 or float16 rounding of each would weigh as much as the result's
// own (64 rows over 32768 bfloat16 keys: 95 us and an error of 0.0017 of the result, which is
// that rounding; with one part 85 us and 0.0023).
//
// What bounds it: a short prefix the chain page, keys, products, parts (4 rows over 500 INT8
// keys 7.1 us and 3.7 of the join); a long one the products and the exponentials, neither of which hides
// behind the other well (64 rows over 131072 bfloat16 keys of 8 heads of 128: per 64 keys and 32 columns
// of a wavefront 1536 cycles of products, some 1900 of vector instructions, 4200 in all).
// 64 rows over 32768 keys and 350 of their own, 32 / 8 heads of 128: bfloat16 over bfloat16 94 us,
// over INT8 90, float16 95; float32 over INT8 98, float16 105 (15 registers spilled), bfloat16
// 147 (one wavefront per SIMD).
// ---------------------------------------------------------------------------
constexpr int kPrefixThreads = 256;
constexpr float kPrefixSlack = 4.0f;
constexpr int kPrefixReads = 4;
constexpr int kHwSlot = 4 | 0 << 6 | 3 << 11;   // s_getreg: hardware register 4 (HW_ID), bits 0 .. 3, the wavefront's slot

template <int HD, int DT, int QP, int PP, int QW>
struct Prefix {
    static constexpr bool BF = DT == DT_BF16;
    static constexpr int ES = DT == DT_I8 ? 1 : 2;
    static constexpr int KG = 4 / QW;                 // wavefronts' groups with keys of their own
    static constexpr int KT = QW == 4 ? 64 : 32;      // keys of a tile
    static constexpr int SUB = KT / 32;
    static constexpr int T = 64 * QW;                 // threads that bring a tile
    static constexpr int KC = HD / 32;                // S products per 16 keys
    static constexpr int VD = HD / 16;                // O products
    static constexpr int COLS = 32 * QW;
    // keys: 8 dimensions of a key at a time
    static constexpr int UK = HD / 8;                 // of a key
    static constexpr int KN = KT * UK / T;            // of a thread
    // values: VN dimensions of 8 keys
    static constexpr int UV = T * 8 / KT;             // of 8 keys
    static constexpr int VN = HD / UV;
    static constexpr int TILE = KT * HD * 2;          // bytes of a tile's keys, or values, in LDS
    static constexpr int BUF = QW == 4 ? 2 : 1;
    static constexpr int PARTS = KG > 1 ? 4 * 32 * (HD + 4) * 4 : 0;   // bytes of O when the wavefronts join
    static constexpr int LDS = std::max(KG * BUF * 2 * TILE, PARTS);

    // where dimensions 8 u .. 8 u + 7 of a tile's key stand: fragment (32 keys, 16-key tile, 32
    // dimensions), lane group u % 4, row m; rows are swapped by u so that a key's pieces, which
    // neighbouring threads write, fall into different banks
    TL_DEV static int key_at(int key, int u) {
        const int sub = key >> 5, t = key >> 2 & 1, m = (key >> 3 & 3) * 4 + (key & 3);
        return (((sub * 2 + t) * KC + (u >> 2)) * 4 + (u & 3)) * 256 + ((m ^ (u & 15)) * 16);
    }
    // where 8 keys (octet of the tile) of dimension d stand: fragment (32 keys, 16 dimensions),
    // lane group octet % 4, row d % 16
    TL_DEV static int value_at(int octet, int d) {
        return (((octet >> 2) * VD + (d >> 4)) * 4 + (octet & 3)) * 256 + (d & 15) * 16;
    }
};

typedef const __attribute__((address_space(4))) int32_t* scalar_table;

// two floats to the 16-bit type, each to nearest
template <bool BF>
TL_DEV int round2(float a, float b) {
    const v2f v = {a, b};
    if constexpr (BF) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(int, __builtin_convertvector(v, b2));
    } else {
        return __builtin_bit_cast(int, __builtin_convertvector(v, h2));
    }
}
// what a pair of 16-bit values leaves of a and b
template <bool BF>
TL_DEV void less2(int w, float& a, float& b) {
    if constexpr (BF) {
        a -= __uint_as_float((unsigned)w << 16);
        b -= __uint_as_float((unsigned)w & 0xFFFF0000u);
    } else {
        const h2 h = __builtin_bit_cast(h2, w);
        a = __builtin_fmaf(-1.0f, (float)h[0], a);
        b = __builtin_fmaf(-1.0f, (float)h[1], b);
    }
}

// W bytes times 8 rows to registers
template <int BYTES>
struct Piece {
    unsigned w[BYTES < 4 ? 1 : BYTES / 4];
    TL_DEV void load(const char* p) {
        if constexpr (BYTES == 2) w[0] = *(const uint16_t*)p;
        else if constexpr (BYTES == 4) w[0] = *(const unsigned*)p;
        else if constexpr (BYTES == 8) {
            const v2i v = *(const v2i*)p;
            w[0] = (unsigned)v[0], w[1] = (unsigned)v[1];
        } else {
            const v4i v = *(const v4i*)p;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = (unsigned)v[i];
        }
    }
};

template <int HD, int DT, int QP, int PP, int QW>
TL_DEV void prefix_run(const PagedAttnArgs& a, const int me, const int workgroups, const int qblocks, char* lds, float (*s_ml)[32][2]) {
    using P = Prefix<HD, DT, QP, PP, QW>;
    constexpr bool BF = P::BF;
    const PagedGeom& geo = a.c.g;
    const int rep = a.n_heads / geo.n_kv;
    const int lane = lane_id(), wave = wave_id(), col = lane & 15, g = lane >> 4;
    const int group = wave / QW, wq = wave % QW, tid = wq * 64 + lane;   // key group, columns, thread of the group

    // workgroup: (KV head, split, column block), column blocks that read the same keys side by
    // side on one XCD
    const int xcd = me % 8, per = workgroups / 8, rem = workgroups % 8;
    const int at = xcd * per + min(xcd, rem) + me / 8;
    const int qb = at % qblocks, split = at / qblocks % a.prefix.splits, kvh = at / qblocks / a.prefix.splits;
    const int len = a.prefix.len;
    const int steps_all = (len + P::KT * P::KG - 1) / (P::KT * P::KG);
    const PagedShare share = paged_share(steps_all, a.prefix.splits);
    const int s0 = share.start(split), s1 = share.start(split + 1);

    const scalar_table table = (scalar_table)(geo.table + (int64_t)a.prefix.seq * geo.table_stride);
    const int last8 = (len - 1) & ~7;
    const int page_mask = (1 << geo.page_shift) - 1;
    const int64_t page_bytes = geo.page_stride * P::ES;
    const int64_t head_bytes = ((int64_t)kvh << geo.page_shift) * (HD * P::ES);
    const char* kbase = (const char*)a.c.k + head_bytes;
    const char* vbase = (const char*)a.c.v + head_bytes;

    // columns of this lane: query head and row (rows that take nothing from here among them, whose q
    // may meanwhile be written over by their results)
    int64_t q_at[2];
    int rows_of[2], head_of[2];
    const int columns = a.rows * rep;   // (below 2^30)
#pragma unroll
    for (int ct = 0; ct < 2; ct++) {
        const int c = min(qb * P::COLS + wq * 32 + ct * 16 + col, columns - 1);
        rows_of[ct] = (int)((unsigned)c / (unsigned)rep);
        head_of[ct] = kvh * rep + c - rows_of[ct] * rep;
        q_at[ct] = (int64_t)rows_of[ct] * a.q_stride + (int64_t)head_of[ct] * HD;
    }
    v4i qf[QP][2][P::KC];
    float cs[2];
#pragma unroll
    for (int ct = 0; ct < 2; ct++) {
        float mx = 0.0f;
        float q[P::KC][8];
#pragma unroll
        for (int c = 0; c < P::KC; c++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const v4f v = load4(a.q, q_at[ct] + (c * 4 + g) * 8 + 4 * h, a.act);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    q[c][4 * h + j] = v[j];
                    mx = fmaxf(mx, fabsf(v[j]));
                }
            }
        float s = a.scale * kLog2e;
        if constexpr (DT == DT_I8) s *= a.c.ks[kvh];
        // the sign of the scale goes to q, so that the largest product has the largest score
        float up = s < 0.0f ? -1.0f : 1.0f;
        s = fabsf(s);
        if constexpr (!BF) {
            mx = pair_max(mx);
            // max |q| in [2^13, 2^14): an infinite, NaN or zero row stays as it is
            const int e = mx > 0.0f && mx < __builtin_inff() ? min(14 - __builtin_amdgcn_frexp_expf(mx), 126) : 0;
            up = __builtin_amdgcn_ldexpf(up, e);
            s = __builtin_amdgcn_ldexpf(s, -e);
        }
        // all scores alike: products of 0, so that a masked one stays minus infinity
        if (s == 0.0f) {
            up = 0.0f;
            s = 1.0f;
        }
        cs[ct] = s;
#pragma unroll
        for (int c = 0; c < P::KC; c++) {
            float rest[8];
#pragma unroll
            for (int j = 0; j < 8; j++) rest[j] = q[c][j] * up;
#pragma unroll
            for (int p = 0; p < QP; p++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    qf[p][ct][c][j] = round2<BF>(rest[2 * j], rest[2 * j + 1]);
                    less2<BF>(qf[p][ct][c][j], rest[2 * j], rest[2 * j + 1]);
                }
        }
    }

    // a tile's pieces on their way: KN times 8 dimensions of a key, VN dimensions of 8 keys
    Piece<8 * P::ES> kr[P::KN];
    Piece<P::VN * P::ES> vr[8];
    // Pages of the next tile to be read, of each of this thread's pieces; those of the keys
    // are the wavefront's, as its keys of one load lie in one group of 8.  They are vector
    // loads: a scalar load in flight makes every LDS read wait for it.
    int32_t k_page[P::KN], v_page;
    int zero;
    asm("v_mov_b32 %0, 0" : "=v"(zero));
    const int32_t* pages = geo.table + (int64_t)a.prefix.seq * geo.table_stride;
    auto k_octet = [&](int j) { return (j * P::T + wq * 64) / P::UK >> 3; };
    const int v_octet = tid / P::UV, v_d = tid % P::UV * P::VN;
    auto look_up = [&](int step) {
        const int key0 = (step * P::KG + group) * P::KT;
#pragma unroll
        for (int j = 0; j < P::KN; j++) k_page[j] = pages[(min(key0 + 8 * k_octet(j), last8) >> geo.page_shift) + zero];
        v_page = pages[min(key0 + 8 * v_octet, last8) >> geo.page_shift];
    };
    uint32_t k_off[P::KN];
#pragma unroll
    for (int j = 0; j < P::KN; j++) {
        const int i = j * P::T + tid;
        k_off[j] = (uint32_t)((i / P::UK % 8) * HD + i % P::UK * 8) * P::ES;
    }
    auto in_pool = [&](int32_t page) { return (unsigned)page < (unsigned)geo.n_pages ? page : 0; };
    auto fetch = [&](int step) {
        const int key0 = (step * P::KG + group) * P::KT;
        // rows behind the last key are read where its eight are
#pragma unroll
        for (int j = 0; j < P::KN; j++) {
            // a base of the wavefront's and a place in its eight rows
            const char* eight = kbase + in_pool(__builtin_amdgcn_readfirstlane(k_page[j])) * page_bytes +
                                (min(key0 + 8 * k_octet(j), last8) & page_mask) * (HD * P::ES);
            kr[j].load(eight + k_off[j]);
        }
        const char* v = vbase + in_pool(v_page) * page_bytes + ((min(key0 + 8 * v_octet, last8) & page_mask) * HD + v_d) * P::ES;
#pragma unroll
        for (int r = 0; r < 8; r++) vr[r].load(v + r * HD * P::ES);
    };
    // groups of 8 of a tile whose page is out of range
    auto lost_of = [&](int step) {
        const int key0 = (step * P::KG + group) * P::KT;
        unsigned bad = 0;
        for (int o = 0; o < P::KT / 8; o++) {
            const int32_t page = table[min(key0 + 8 * o, last8) >> geo.page_shift];
            bad |= (unsigned)page >= (unsigned)geo.n_pages ? 1u << o : 0u;
        }
        return bad;
    };
    char* const k_lds = lds + group * (P::BUF * 2 * P::TILE);
    auto keep = [&](int step, bool whole, unsigned bad) {
        char* kl = k_lds + (P::BUF == 2 ? (step & 1) * 2 * P::TILE : 0);
        char* vl = kl + P::TILE;
#pragma unroll
        for (int j = 0; j < P::KN; j++) {
            const int i = j * P::T + tid, key = i / P::UK, u = i % P::UK;
            v4i w;
            if constexpr (DT == DT_I8) {
                const unsigned w0 = kr[j].w[0], w1 = kr[j].w[1];
                w = v4i{i8_pair_f16(__builtin_amdgcn_perm(0u, w0, 0x0C010C00u)), i8_pair_f16(__builtin_amdgcn_perm(0u, w0, 0x0C030C02u)),
                        i8_pair_f16(__builtin_amdgcn_perm(0u, w1, 0x0C010C00u)), i8_pair_f16(__builtin_amdgcn_perm(0u, w1, 0x0C030C02u))};
            } else {
                w = v4i{(int)kr[j].w[0], (int)kr[j].w[1], (int)kr[j].w[2], (int)kr[j].w[3]};
            }
            *(v4i*)(kl + P::key_at(key, u)) = w;
        }
        if (!whole) {   // values of keys behind the last one and of lost pages are zero, as 0 x NaN is NaN
            asm volatile("");
            const int left = bad >> v_octet & 1 ? 0 : len - ((step * P::KG + group) * P::KT + 8 * v_octet);
#pragma unroll
            for (int r = 0; r < 8; r++)
#pragma unroll
                for (unsigned& w : vr[r].w) w = r < left ? w : 0u;
        }
#pragma unroll
        for (int i = 0; i < P::VN; i++) {
            v4i w;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const unsigned x = vr[2 * r].w[i * P::ES / 4], y = vr[2 * r + 1].w[i * P::ES / 4];
                if constexpr (DT == DT_I8) w[r] = i8_pair_f16(__builtin_amdgcn_perm(y, x, 0x0C040C00u + 0x00010001u * (unsigned)(i & 3)));
                else w[r] = (int)__builtin_amdgcn_perm(y, x, i & 1 ? 0x07060302u : 0x05040100u);
            }
            *(v4i*)(vl + P::value_at(v_octet, v_d + i)) = w;
        }
    };

    float m[2] = {-__builtin_inff(), -__builtin_inff()}, l[2] = {0.0f, 0.0f};   // m: of products; l: this lane's keys
    v4f o[P::VD][2];
#pragma unroll
    for (int j = 0; j < P::VD; j++) o[j][0] = o[j][1] = v4f{0, 0, 0, 0};

    // whether a page of this split is out of range: looked at once, so that no tile has to
    bool any_lost = false;
    {
        const int first = (s0 * P::KG * P::KT) >> geo.page_shift, last = (min(s1 * P::KG * P::KT, len) - 1) >> geo.page_shift;
        for (int p = first + lane; p <= last; p += 64) any_lost |= (unsigned)table[p] >= (unsigned)geo.n_pages;
        any_lost = __builtin_amdgcn_ballot_w64(any_lost) != 0;
    }
    // Two wavefronts on a SIMD that take turns at equal rights stay in step, both at their
    // exponentials and then both at their products; so one of them, by its slot, goes first
    // (64 rows over 131072 keys of 8 heads of 128: 259 us, 266 without).
    if (__builtin_amdgcn_s_getreg(kHwSlot) & 1) __builtin_amdgcn_s_setprio(1);
    if (s0 < s1) {
        look_up(s0);
        fetch(s0);
        look_up(min(s0 + 1, s1 - 1));
    }
    for (int step = s0; step < s1; step++) {
        if constexpr (P::BUF == 1) __builtin_amdgcn_wave_barrier();
        const int key0 = (step * P::KG + group) * P::KT;
        unsigned bad_now = 0;
        if (any_lost) bad_now = lost_of(step);
        const bool whole = key0 + P::KT <= len && bad_now == 0;
        keep(step, whole, bad_now);
        if constexpr (P::BUF == 2) __syncthreads();
        else __builtin_amdgcn_wave_barrier();
        if (step + 1 < s1) {
            fetch(step + 1);
            look_up(min(step + 2, s1 - 1));
        }
        const char* kl = k_lds + (P::BUF == 2 ? (step & 1) * 2 * P::TILE : 0);
        const char* vl = kl + P::TILE;
        // Operands are read kPrefixReads products early; left to itself the compiler reads each
        // just before its products and waits for it.
        v4f s[P::SUB][2][2];
        {
            constexpr int N = P::SUB * 2 * P::KC;
            v4i kk[kPrefixReads];
            auto read = [&](int i) {
                const int u = i % P::KC * 4 + g;
                kk[i % kPrefixReads] = *(const v4i*)(kl + (i * 4 + g) * 256 + ((col ^ (u & 15)) * 16));
            };
#pragma unroll
            for (int i = 0; i < kPrefixReads; i++) read(i);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int sub = i / (2 * P::KC), t = i / P::KC % 2, c = i % P::KC;
                if (c == 0) s[sub][t][0] = s[sub][t][1] = v4f{0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < QP; p++)
#pragma unroll
                    for (int ct = 0; ct < 2; ct++) s[sub][t][ct] = mfma32<BF>(kk[i % kPrefixReads], qf[p][ct][c], s[sub][t][ct]);
                __builtin_amdgcn_sched_barrier(0);
                if (i + kPrefixReads < N) read(i + kPrefixReads);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (!whole) {
            asm volatile("");    // a branch, no selects in every tile
            unsigned in = 0;     // keys 32 sub + 8 g + j: bit 8 sub + j
#pragma unroll
            for (int sub = 0; sub < P::SUB; sub++) {
                const int left = len - (key0 + 32 * sub + 8 * g);
                const unsigned mine = left >= 8 ? 0xFFu : left <= 0 ? 0u : (1u << left) - 1;
                if (!(bad_now >> (4 * sub + g) & 1)) in |= mine << (8 * sub);
            }
#pragma unroll
            for (int sub = 0; sub < P::SUB; sub++)
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int ct = 0; ct < 2; ct++)
                        if (!(in >> (8 * sub + j) & 1)) s[sub][j >> 2][ct][j & 3] = -__builtin_inff();
        }
        v4i pf[P::SUB][PP][2];
#pragma unroll
        for (int ct = 0; ct < 2; ct++) {
            float mt = -__builtin_inff();
#pragma unroll
            for (int sub = 0; sub < P::SUB; sub++)
#pragma unroll
                for (int j = 0; j < 8; j++) mt = fmaxf(mt, s[sub][j >> 2][ct][j & 3]);
            mt = pair_max(mt);
            // A column's sums are scaled anew only where a score leaves them by kPrefixSlack: a fresh
            // maximum, of which most tiles have one among 16 columns, alone does not.  The other
            // columns take a factor of 1: a row's bits do not depend on what stands in the others.
            const bool leaves = mt * cs[ct] > m[ct] * cs[ct] + kPrefixSlack;
            if (__builtin_amdgcn_ballot_w64(leaves) != 0) {
                asm volatile("");
                const float mn = leaves ? mt : m[ct];
                const float al = !leaves ? 1.0f : m[ct] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m[ct] - mn) * cs[ct]);
                m[ct] = mn;
                l[ct] *= al;
#pragma unroll
                for (int j = 0; j < P::VD; j++) o[j][ct] *= al;
            }
            // p 2^14 over float16, so that the parts of small probabilities stay normal; 2^10 of it
            // here, as a score may lie kPrefixSlack above m
            const float off = (m[ct] == -__builtin_inff() ? 0.0f : m[ct] * cs[ct]) - (BF ? 0.0f : 14.0f - kPrefixSlack);
#pragma unroll
            for (int sub = 0; sub < P::SUB; sub++) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][j >> 2][ct][j & 3], cs[ct], -off));
                    l[ct] += p[j];
                }
#pragma unroll
                for (int part = 0; part < PP; part++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        pf[sub][part][ct][j] = round2<BF>(p[2 * j], p[2 * j + 1]);
                        if (part + 1 < PP) less2<BF>(pf[sub][part][ct][j], p[2 * j], p[2 * j + 1]);
                    }
            }
        }
        {
            constexpr int N = P::SUB * P::VD;
            v4i vv[kPrefixReads];
            auto read = [&](int i) { vv[i % kPrefixReads] = *(const v4i*)(vl + (i * 4 + g) * 256 + col * 16); };
#pragma unroll
            for (int i = 0; i < kPrefixReads; i++) read(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int sub = i / P::VD, j = i % P::VD;
#pragma unroll
                for (int part = 0; part < PP; part++)
#pragma unroll
                    for (int ct = 0; ct < 2; ct++) o[j][ct] = mfma32<BF>(vv[i % kPrefixReads], pf[sub][part][ct], o[j][ct]);
                __builtin_amdgcn_sched_barrier(0);
                if (i + kPrefixReads < N) read(i + kPrefixReads);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if (a.fault && any_lost) *a.fault = 1;

    // m in units of the exponent, l over the lane groups, values' scale
    const float sv = DT == DT_I8 ? a.c.vs[kvh] : 1.0f;
#pragma unroll
    for (int ct = 0; ct < 2; ct++) {
        // (2^14 of the probabilities over float16, as the other kernel's parts)
        m[ct] = m[ct] == -__builtin_inff() ? m[ct] : m[ct] * cs[ct] + (BF ? 0.0f : kPrefixSlack);
        l[ct] += lane_xor<16>(l[ct]);
        l[ct] += lane_xor<32>(l[ct]);
    }
    if constexpr (P::KG == 1) {
#pragma unroll
        for (int ct = 0; ct < 2; ct++) {
            if (qb * P::COLS + wq * 32 + ct * 16 + col >= columns) continue;
            const int64_t part = prefix_part(a, split, rows_of[ct], head_of[ct]);
            if (g == 0) *(v2f*)(a.prefix.ml + 2 * part) = v2f{m[ct], l[ct]};
#pragma unroll
            for (int j = 0; j < P::VD; j++) *(v4f*)(a.prefix.o + part * HD + 16 * j + 4 * g) = o[j][ct] * sv;
        }
    } else {
        __syncthreads();
        float* mine = (float*)(lds + wave * (32 * (HD + 4) * 4));
#pragma unroll
        for (int ct = 0; ct < 2; ct++) {
            if (g == 0) {
                s_ml[wave][ct * 16 + col][0] = m[ct];
                s_ml[wave][ct * 16 + col][1] = l[ct];
            }
#pragma unroll
            for (int j = 0; j < P::VD; j++) *(v4f*)(mine + (ct * 16 + col) * (HD + 4) + 16 * j + 4 * g) = o[j][ct];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * HD / 4; i += kPrefixThreads) {
            const int c = i / (HD / 4), d = (i - c * (HD / 4)) * 4;
            const int column = qb * P::COLS + c;
            if (column >= columns) continue;
            float mm = s_ml[0][c][0];
#pragma unroll
            for (int w = 1; w < 4; w++) mm = fmaxf(mm, s_ml[w][c][0]);
            const float off = mm == -__builtin_inff() ? 0.0f : mm;
            float ll = 0.0f;
            v4f acc = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float e = __builtin_amdgcn_exp2f(s_ml[w][c][0] - off);
                ll += e * s_ml[w][c][1];
                acc += e * *(const v4f*)((const float*)(lds + w * (32 * (HD + 4) * 4)) + c * (HD + 4) + d);
            }
            const int row = (int)((unsigned)column / (unsigned)rep);
            const int64_t part = prefix_part(a, split, row, kvh * rep + column - row * rep);
            if (d == 0) *(v2f*)(a.prefix.ml + 2 * part) = v2f{mm, ll};
            *(v4f*)(a.prefix.o + part * HD + d) = acc * sv;
        }
    }
}

template <int HD, int DT, int QP, int PP, int QW>
__global__ __launch_bounds__(kPrefixThreads, QP == 3 ? 1 : 2) void shared_attention_kernel(PagedAttnArgs a, SharedRoles roles, int qblocks) {
    extern __shared__ __align__(16) char lds[];
    __shared__ float s_ml[4][32][2];
    int at;
    if (roles.is_own(blockIdx.x, at)) attention_run<HD, DT, QP == 3, true>(a, at, roles.own, *(AttnShared<HD, DT, QP == 3>*)lds);
    else prefix_run<HD, DT, QP, PP, QW>(a, at, roles.prefix, qblocks, lds, s_ml);
}

// What the rows' own keys and the prefix left of a query head, joined: workgroup (row, head,
// or several heads where there are few parts), `lanes` parts of a head side by side.
template <int HD>
__global__ __launch_bounds__(kPrefixThreads) void shared_join_kernel(PagedAttnArgs a, int own_workgroups, int lanes) {
    constexpr int Q = HD / 4, W = kPrefixThreads / Q, AHEAD = 4;
    __shared__ float s_acc[W][HD], s_l[W], s_m[W];
    const PagedGeom& geo = a.c.g;
    const int rep = a.n_heads / geo.n_kv, blocks = (rep + 7) >> 3;
    const int q = threadIdx.x % Q, slot = threadIdx.x / Q, s = slot % lanes;
    const int row = blockIdx.x, head = blockIdx.y * (W / lanes) + slot / lanes;
    const int pos = a.row_pos[row];
    if (paged_row_kind(geo, a.row_seq ? a.row_seq[row] : row, pos) != PAGED_ROW_OK) return;
    const bool adds = shared_adds(a.prefix.len, pos);
    const int tiles = shared_tiles(a.prefix.len, pos);
    const PagedShare share = paged_share(a.prefix.starts[a.rows], own_workgroups);
    const int kvh = min(head, a.n_heads - 1) / rep, h = min(head, a.n_heads - 1) - kvh * rep;
    const int32_t unit = a.prefix.starts[row] + (kvh * blocks + (h >> 3)) * tiles;
    const int w0 = share.owner(unit), w1 = share.owner(unit + tiles - 1);
    // the prefix's parts, then the own keys': whole, of no keys none, or in parts
    const int slots = adds ? a.prefix.splits + (w0 == w1 && pos + 1 > a.prefix.len) : 0;
    const int parts = head < a.n_heads ? slots + (w0 == w1 ? 0 : w1 - w0 + 1) : 0;
    float m = -__builtin_inff(), l = 0.0f;
    v4f acc = {0, 0, 0, 0};
    for (int p0 = s; p0 < parts; p0 += AHEAD * lanes) {
        v2f ml[AHEAD];
        v4f o[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int p = min(p0 + j * lanes, parts - 1);
            const float *from_o, *from_ml;
            if (p < slots) {
                const int64_t part = prefix_part(a, p, row, head);
                from_o = a.prefix.o + part * HD;
                from_ml = a.prefix.ml + 2 * part;
            } else {
                const int part = paged_part(share, w0 + p - slots, unit);
                from_o = part_o<HD>(a, part) + (h & 7) * HD;
                from_ml = part_ml<HD>(a, part, own_workgroups) + 2 * (h & 7);
            }
            o[j] = *(const v4f*)(from_o + 4 * q);
            ml[j] = *(const v2f*)from_ml;
            if (p0 + j * lanes >= parts) ml[j][0] = -__builtin_inff();
        }
        float mm = m;
#pragma unroll
        for (int j = 0; j < AHEAD; j++) mm = fmaxf(mm, ml[j][0]);
        const float off = mm == -__builtin_inff() ? 0.0f : mm;
        const float keep = __builtin_amdgcn_exp2f(m - off);
        m = mm;
        l *= keep;
        acc *= keep;
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const float e = __builtin_amdgcn_exp2f(ml[j][0] - off);
            l += e * ml[j][1];
            acc += e * o[j];
        }
    }
    *(v4f*)&s_acc[slot][4 * q] = acc;
    if (q == 0) {
        s_l[slot] = l;
        s_m[slot] = m;
    }
    __syncthreads();
    if (s != 0 || parts == 0) return;
    float mm = m;
    for (int i = 1; i < lanes; i++) mm = fmaxf(mm, s_m[slot + i]);
    const float off = mm == -__builtin_inff() ? 0.0f : mm;
    const float keep = __builtin_amdgcn_exp2f(m - off);
    l *= keep;
    acc *= keep;
    for (int i = 1; i < lanes; i++) {
        const float e = __builtin_amdgcn_exp2f(s_m[slot + i] - off);
        l += e * s_l[slot + i];
        acc += e * *(const v4f*)&s_acc[slot + i][4 * q];
    }
    store4(a.out, (int64_t)row * a.out_stride + (int64_t)head * HD + 4 * q, a.act, acc / l);
}

// Calls f(instance) with the instance for a's types: parts of q and of the probabilities
template <int HD, int DT, int QP, int PP, int QW>
struct Instance {
    static constexpr auto kernel = shared_attention_kernel<HD, DT, QP, PP, QW>;
    static constexpr int LDS = std::max<int>(Prefix<HD, DT, QP, PP, QW>::LDS, sizeof(AttnShared<HD, DT, QP == 3>));
};
template <int HD, int QW, typename F>
hipError_t with_types(int dtype, int act, F f) {
    const bool f32 = act == DT_F32;
    if (dtype == DT_BF16) return act == DT_BF16 ? f(Instance<HD, DT_BF16, 1, 2, QW>{}) : f(Instance<HD, DT_BF16, 3, 3, QW>{});
    if (dtype == DT_F16) return f32 ? f(Instance<HD, DT_F16, 2, 2, QW>{}) : f(Instance<HD, DT_F16, 1, 2, QW>{});
    return f32 ? f(Instance<HD, DT_I8, 2, 2, QW>{}) : f(Instance<HD, DT_I8, 1, 2, QW>{});
}
template <typename F>
hipError_t with_instance(int hd, int qw, int dtype, int act, F f) {
    if (hd == 64) return qw == 1 ? with_types<64, 1>(dtype, act, f) : with_types<64, 4>(dtype, act, f);
    return qw == 1 ? with_types<128, 1>(dtype, act, f) : with_types<128, 4>(dtype, act, f);
}

}  // namespace

hipError_t launch_shared_attention(hipStream_t s, const PagedAttnArgs& a) {
    const PrefixPlan p = prefix_plan(a.rows, a.n_heads, a.c.g.n_kv, a.prefix.len);
    const SharedRoles roles{p.grid, paged_attention_workgroups(a.c, a.rows, a.n_heads)};
    const hipError_t e = with_instance(a.c.g.head_dim, p.qw, a.c.dtype, a.act, [&](auto i) {
        using I = decltype(i);
        TL_KLAUNCH(I::kernel, dim3(roles.prefix + roles.own), dim3(kPrefixThreads), I::LDS, s, a, roles, p.qblocks);
        return hipGetLastError();
    });
    if (e != hipSuccess) return e;
    const int side = kPrefixThreads / (a.c.g.head_dim / 4);   // parts that a workgroup takes side by side
    const int lanes = shared_join_lanes(side, p.splits, roles.own, (int64_t)a.rows * a.n_heads);
    const dim3 grid(a.rows, (a.n_heads + side / lanes - 1) / (side / lanes));
    if (a.c.g.head_dim == 64) TL_KLAUNCH((shared_join_kernel<64>), grid, dim3(kPrefixThreads), 0, s, a, roles.own, lanes);
    else TL_KLAUNCH((shared_join_kernel<128>), grid, dim3(kPrefixThreads), 0, s, a, roles.own, lanes);
    return hipGetLastError();
}

hipError_t init_prefix_kernels() {
    hipError_t e = hipSuccess;
    for (int hd : {64, 128})
        for (int qw : {1, 4})
            for (int dtype : {DT_I8, DT_BF16, DT_F16})
                for (int act : {DT_F32, DT_BF16})
                    if (e == hipSuccess)
                        e = with_instance(hd, qw, dtype, act, [](auto i) {
                            using I = decltype(i);
                            return hipFuncSetAttribute((const void*)I::kernel, hipFuncAttributeMaxDynamicSharedMemorySize, I::LDS);
                        });
    return e;
}

size_t paged_shared_scratch(const PagedCache& c, int32_t rows, int32_t n_heads, int32_t len) {
    if (rows <= 0) return 0;
    const size_t own = paged_attention_scratch(c, rows, n_heads);
    if (len <= 0) return own;
    const PrefixPlan p = prefix_plan(rows, n_heads, c.g.n_kv, len);
    return (own + 15) / 16 * 16 + ((size_t)(p.splits + 1) * rows * n_heads * (c.g.head_dim + 2) + rows + 1) * sizeof(float);
}

void paged_shared_places(PagedAttnArgs& a) {
    if (a.prefix.len <= 0 || a.rows <= 0) return;
    const PrefixPlan p = prefix_plan(a.rows, a.n_heads, a.c.g.n_kv, a.prefix.len);
    a.prefix.splits = p.splits;
    a.prefix.o = (float*)((char*)a.scratch + (paged_attention_scratch(a.c, a.rows, a.n_heads) + 15) / 16 * 16);
    a.prefix.ml = a.prefix.o + (int64_t)(p.splits + 1) * a.rows * a.n_heads * a.c.g.head_dim;
    a.prefix.starts = (int32_t*)(a.prefix.ml + (int64_t)(p.splits + 1) * a.rows * a.n_heads * 2);
}

}  // namespace tl
