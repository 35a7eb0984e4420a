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
// The keys are split over workgroups; each leaves O, m and l of its columns in scratch,
// which the kernel of the rows' own keys adds to those (paged_attention_kernel).
//
// Precision: q enters in QP 16-bit parts and the probabilities in PP, as many as it takes:
// of 16-bit rows q is exact in one (float16 holds a bfloat16 scaled to its row); float32 rows
// take two float16 parts (within 2^-23) or three bfloat16 ones (whole).  Probabilities of 16-bit rows take
// two parts, as one bfloat16 or float16 rounding of each would weigh as much as the result's own.
// ---------------------------------------------------------------------------
constexpr int kPrefixThreads = 256;

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
__global__ __launch_bounds__(kPrefixThreads, QP == 3 ? 1 : 2) void paged_prefix_kernel(PagedAttnArgs a, int qblocks) {
    using P = Prefix<HD, DT, QP, PP, QW>;
    constexpr bool BF = P::BF;
    extern __shared__ __align__(16) char lds[];
    __shared__ float s_ml[4][32][2];
    const PagedGeom& geo = a.c.g;
    const int rep = a.n_heads / geo.n_kv;
    const int lane = lane_id(), wave = wave_id(), col = lane & 15, g = lane >> 4;
    const int group = wave / QW, wq = wave % QW, tid = wq * 64 + lane;   // key group, columns, thread of the group

    // workgroup: (KV head, split, column block), column blocks that read the same keys side by
    // side on one XCD
    const int all = gridDim.x, xcd = blockIdx.x % 8, per = all / 8, rem = all % 8;
    const int at = xcd * per + min(xcd, rem) + blockIdx.x / 8;
    const int qb = at % qblocks, split = at / qblocks % a.prefix.splits, kvh = at / qblocks / a.prefix.splits;
    const int len = a.prefix.len;
    const int steps_all = (len + P::KT * P::KG - 1) / (P::KT * P::KG);
    const int s0 = (int)((int64_t)steps_all * split / a.prefix.splits), s1 = (int)((int64_t)steps_all * (split + 1) / a.prefix.splits);

    const scalar_table table = (scalar_table)(geo.table + (int64_t)a.prefix.seq * geo.table_stride);
    const int last8 = (len - 1) & ~7;
    const int page_mask = (1 << geo.page_shift) - 1;
    const int64_t page_bytes = geo.page_stride * P::ES;
    const int64_t head_bytes = ((int64_t)kvh << geo.page_shift) * (HD * P::ES);
    const char* kbase = (const char*)a.c.k + head_bytes;
    const char* vbase = (const char*)a.c.v + head_bytes;

    // columns of this lane: query head and row
    int64_t q_at[2];
    int rows_of[2], head_of[2];
    const int64_t columns = (int64_t)a.rows * rep;
#pragma unroll
    for (int ct = 0; ct < 2; ct++) {
        const int64_t c = std::min<int64_t>((int64_t)qb * P::COLS + wq * 32 + ct * 16 + col, columns - 1);
        rows_of[ct] = (int)(c / rep);
        head_of[ct] = kvh * rep + (int)(c - (int64_t)rows_of[ct] * rep);
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
                    unsigned w[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        w[i] = BF ? to_bf16(rest[2 * j + i]) : to_f16(rest[2 * j + i]);
                        rest[2 * j + i] -= BF ? bf16_bits(w[i]) : f16_bits(w[i]);
                    }
                    qf[p][ct][c][j] = (int)(w[0] | w[1] << 16);
                }
        }
    }

    // a tile's pieces on their way: KN times 8 dimensions of a key, VN dimensions of 8 keys
    Piece<8 * P::ES> kr[P::KN];
    Piece<P::VN * P::ES> vr[8];
    int32_t pages[P::KT / 8];      // of the next tile to be read
    unsigned bad = 0;              // octets of the tile in registers whose page is out of range
    bool any_bad = false;
    auto look_up = [&](int step) {
        const int key0 = (step * P::KG + group) * P::KT;
#pragma unroll
        for (int o = 0; o < P::KT / 8; o++) pages[o] = table[min(key0 + 8 * o, last8) >> geo.page_shift];
    };
    const int v_octet = tid / P::UV, v_d = tid % P::UV * P::VN;
    auto fetch = [&](int step) {
        const int key0 = (step * P::KG + group) * P::KT;
        bad = 0;
#pragma unroll
        for (int o = 0; o < P::KT / 8; o++)
            if ((unsigned)pages[o] >= (unsigned)geo.n_pages) {
                bad |= 1u << o;
                pages[o] = 0;
            }
        // rows behind the last key are read where its eight are
#pragma unroll
        for (int j = 0; j < P::KN; j++) {
            const int i = j * P::T + tid, key = i / P::UK, u = i % P::UK;
            const int octet = __builtin_amdgcn_readfirstlane(key >> 3);   // the wavefront's keys lie in one
            int32_t page = pages[0];
#pragma unroll
            for (int o = 1; o < P::KT / 8; o++) page = octet == o ? pages[o] : page;
            const int k = min(key0 + 8 * octet, last8) + (key & 7);
            kr[j].load(kbase + page * page_bytes + ((k & page_mask) * HD + 8 * u) * P::ES);
        }
        int32_t page = pages[0];
#pragma unroll
        for (int o = 1; o < P::KT / 8; o++) page = v_octet == o ? pages[o] : page;
        const char* v = vbase + page * page_bytes + ((min(key0 + 8 * v_octet, last8) & page_mask) * HD + v_d) * P::ES;
#pragma unroll
        for (int r = 0; r < 8; r++) vr[r].load(v + r * HD * P::ES);
    };
    char* const k_lds = lds + group * (P::BUF * 2 * P::TILE);
    auto keep = [&](int step) {
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
        // values of keys behind the last one and of pages out of range are zero, as 0 x NaN is NaN
        const int left = len - ((step * P::KG + group) * P::KT + 8 * v_octet);
        const bool lost = bad >> v_octet & 1;
#pragma unroll
        for (int i = 0; i < P::VN; i++) {
            v4i w;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const unsigned x = vr[2 * r].w[i * P::ES / 4], y = vr[2 * r + 1].w[i * P::ES / 4];
                unsigned pair;
                if constexpr (DT == DT_I8) pair = (unsigned)i8_pair_f16(__builtin_amdgcn_perm(y, x, 0x0C040C00u + 0x00010001u * (unsigned)(i & 3)));
                else pair = __builtin_amdgcn_perm(y, x, i & 1 ? 0x07060302u : 0x05040100u);
                if (left < 2 * r + 2) pair = left == 2 * r + 1 ? pair & 0xFFFFu : 0u;
                w[r] = lost ? 0 : (int)pair;
            }
            *(v4i*)(vl + P::value_at(v_octet, v_d + i)) = w;
        }
    };

    float m[2] = {-__builtin_inff(), -__builtin_inff()}, l[2] = {0.0f, 0.0f};   // m: of products; l: this lane's keys
    v4f o[P::VD][2];
#pragma unroll
    for (int j = 0; j < P::VD; j++) o[j][0] = o[j][1] = v4f{0, 0, 0, 0};

    if (s0 < s1) {
        look_up(s0);
        fetch(s0);
        look_up(min(s0 + 1, s1 - 1));
    }
    for (int step = s0; step < s1; step++) {
        if constexpr (P::BUF == 1) __builtin_amdgcn_wave_barrier();
        keep(step);
        const unsigned bad_now = bad;
        if constexpr (P::BUF == 2) __syncthreads();
        else __builtin_amdgcn_wave_barrier();
        if (step + 1 < s1) {
            fetch(step + 1);
            look_up(min(step + 2, s1 - 1));
        }
        const char* kl = k_lds + (P::BUF == 2 ? (step & 1) * 2 * P::TILE : 0);
        const char* vl = kl + P::TILE;
        const int key0 = (step * P::KG + group) * P::KT;
        v4f s[P::SUB][2][2];
#pragma unroll
        for (int sub = 0; sub < P::SUB; sub++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                s[sub][t][0] = s[sub][t][1] = v4f{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < P::KC; c++) {
                    const int u = c * 4 + g;
                    const v4i kk = *(const v4i*)(kl + (((sub * 2 + t) * P::KC + c) * 4 + g) * 256 + ((col ^ (u & 15)) * 16));
#pragma unroll
                    for (int p = 0; p < QP; p++)
#pragma unroll
                        for (int ct = 0; ct < 2; ct++) s[sub][t][ct] = mfma32<BF>(kk, qf[p][ct][c], s[sub][t][ct]);
                }
            }
        const bool whole = key0 + P::KT <= len && bad_now == 0;
        any_bad |= bad_now != 0;
        unsigned in = 0xFFFFu;   // keys 32 sub + 8 g + j: bit 8 sub + j
        if (!whole) {
            in = 0;
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
            if (__builtin_amdgcn_ballot_w64(mt > m[ct]) != 0) {
                const float mn = fmaxf(m[ct], mt);
                const float al = m[ct] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m[ct] - mn) * cs[ct]);
                m[ct] = mn;
                l[ct] *= al;
#pragma unroll
                for (int j = 0; j < P::VD; j++) o[j][ct] *= al;
            }
            // p 2^14, so that the float16 parts of small probabilities stay normal
            const float off = (m[ct] == -__builtin_inff() ? 0.0f : m[ct] * cs[ct]) - (BF ? 0.0f : 14.0f);
#pragma unroll
            for (int sub = 0; sub < P::SUB; sub++) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][j >> 2][ct][j & 3], cs[ct], -off));
                    if (!whole) p[j] = in >> (8 * sub + j) & 1 ? p[j] : 0.0f;
                    l[ct] += p[j];
                }
#pragma unroll
                for (int part = 0; part < PP; part++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        unsigned w[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            w[i] = BF ? to_bf16(p[2 * j + i]) : to_f16(p[2 * j + i]);
                            if (part + 1 < PP) p[2 * j + i] -= BF ? bf16_bits(w[i]) : f16_bits(w[i]);
                        }
                        pf[sub][part][ct][j] = (int)(w[0] | w[1] << 16);
                    }
            }
        }
#pragma unroll
        for (int sub = 0; sub < P::SUB; sub++)
#pragma unroll
            for (int j = 0; j < P::VD; j++) {
                const v4i vv = *(const v4i*)(vl + ((sub * P::VD + j) * 4 + g) * 256 + col * 16);
#pragma unroll
                for (int part = 0; part < PP; part++)
#pragma unroll
                    for (int ct = 0; ct < 2; ct++) o[j][ct] = mfma32<BF>(vv, pf[sub][part][ct], o[j][ct]);
            }
    }
    if (a.fault && any_bad) *a.fault = 1;

    // m in units of the exponent, l over the lane groups, values' scale
    const float sv = DT == DT_I8 ? a.c.vs[kvh] : 1.0f;
#pragma unroll
    for (int ct = 0; ct < 2; ct++) {
        m[ct] = m[ct] == -__builtin_inff() ? m[ct] : m[ct] * cs[ct];
        l[ct] += lane_xor<16>(l[ct]);
        l[ct] += lane_xor<32>(l[ct]);
    }
    if constexpr (P::KG == 1) {
#pragma unroll
        for (int ct = 0; ct < 2; ct++) {
            if ((int64_t)qb * P::COLS + wq * 32 + ct * 16 + col >= columns) continue;
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
            const int64_t column = (int64_t)qb * P::COLS + c;
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
            const int row = (int)(column / rep);
            const int64_t part = prefix_part(a, split, row, kvh * rep + (int)(column - (int64_t)row * rep));
            if (d == 0) *(v2f*)(a.prefix.ml + 2 * part) = v2f{mm, ll};
            *(v4f*)(a.prefix.o + part * HD + d) = acc * sv;
        }
    }
}

// Calls f(instance) with the instance for a's types: parts of q and of the probabilities
template <int HD, int DT, int QP, int PP, int QW>
struct Instance {
    using P = Prefix<HD, DT, QP, PP, QW>;
    static constexpr auto kernel = paged_prefix_kernel<HD, DT, QP, PP, QW>;
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

hipError_t launch_paged_prefix(hipStream_t s, const PagedAttnArgs& a) {
    const PrefixPlan p = prefix_plan(a.rows, a.n_heads, a.c.g.n_kv, a.prefix.len);
    return with_instance(a.c.g.head_dim, p.qw, a.c.dtype, a.act, [&](auto i) {
        using I = decltype(i);
        TL_KLAUNCH(I::kernel, dim3(p.grid), dim3(kPrefixThreads), I::P::LDS, s, a, p.qblocks);
        return hipGetLastError();
    });
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
                            return hipFuncSetAttribute((const void*)I::kernel, hipFuncAttributeMaxDynamicSharedMemorySize, I::P::LDS);
                        });
    return e;
}

size_t paged_shared_scratch(const PagedCache& c, int32_t rows, int32_t n_heads, int32_t len) {
    if (rows <= 0) return 0;
    const size_t own = paged_attention_scratch(c, rows, n_heads);
    if (len <= 0) return own;
    const PrefixPlan p = prefix_plan(rows, n_heads, c.g.n_kv, len);
    return (own + 15) / 16 * 16 + (size_t)p.splits * rows * n_heads * (c.g.head_dim + 4) * sizeof(float);
}

void paged_shared_places(PagedAttnArgs& a) {
    if (a.prefix.len <= 0 || a.rows <= 0) return;
    const PrefixPlan p = prefix_plan(a.rows, a.n_heads, a.c.g.n_kv, a.prefix.len);
    a.prefix.splits = p.splits;
    a.prefix.o = (float*)((char*)a.scratch + (paged_attention_scratch(a.c, a.rows, a.n_heads) + 15) / 16 * 16);
    a.prefix.ml = a.prefix.o + (int64_t)p.splits * a.rows * a.n_heads * a.c.g.head_dim;
}

}  // namespace tl
