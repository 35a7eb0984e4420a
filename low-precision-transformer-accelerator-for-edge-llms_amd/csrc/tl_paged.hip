// tl_paged.hip -- the paged KV cache: append with rotation, and the attention of
// one query row per token over it.
#include <algorithm>

#include "tl_rows.h"

namespace tl {
namespace {

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
// the cache.
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

__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    const PagedGeom& g = a.c.g;
    const int row = blockIdx.x;
    const int seq = a.row_seq ? a.row_seq[row] : row;
    const int pos = a.row_pos[row];
    const PagedRow kind = paged_row_kind(g, seq, pos);
    if (kind == PAGED_ROW_PADDING) return;
    // a position needs its rotation and, for k and v, its page
    const int page = kind == PAGED_ROW_OK && pos >= 0 && pos < a.n_pos ? paged_page(g, seq, pos) : -1;
    if (page < 0) {
        if (a.fault && threadIdx.x == 0 && blockIdx.y == 0) *a.fault = 1;
        return;
    }
    const int hd = g.head_dim, half = hd >> 1, quads = half >> 2;
    const int n_rot = (a.n_heads + g.n_kv) * quads;
    const int u = blockIdx.y * 256 + threadIdx.x;
    const int64_t in = (int64_t)row * a.qkv_stride;
    if (u < n_rot) {
        const int head = u / quads, d = (u - head * quads) * 4;
        if (head < a.n_heads && !a.q_out) return;
        const int64_t at = in + (int64_t)head * hd + d;
        const v4f x1 = load4(a.qkv, at, a.act), x2 = load4(a.qkv, at + half, a.act);
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
            store4(a.q_out, to, a.act, y1);
            store4(a.q_out, to + half, a.act, y2);
        } else {
            const int kvh = head - a.n_heads;
            const float sk = a.c.dtype == DT_I8 ? a.c.ks[kvh] : 1.0f;
            const int64_t to = paged_row(g, page, kvh, pos) + d;
            cache_store4(a.c.k, to, a.c.dtype, y1, sk);
            cache_store4(a.c.k, to + half, a.c.dtype, y2, sk);
        }
        return;
    }
    const int w = (u - n_rot) * 8;
    if (w >= g.n_kv * hd) return;
    const int kvh = w / hd, d = w - kvh * hd;
    const int64_t at = in + (int64_t)(a.n_heads + g.n_kv) * hd + w;
    const float sv = a.c.dtype == DT_I8 ? a.c.vs[kvh] : 1.0f;
    const int64_t to = paged_row(g, page, kvh, pos) + d;
    cache_store4(a.c.v, to, a.c.dtype, load4(a.qkv, at, a.act), sv);
    cache_store4(a.c.v, to + 4, a.c.dtype, load4(a.qkv, at + 4, a.act), sv);
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
// p in the 16-bit type, one with the rest.  Their sums restore about 22 bits
// (float16) or 16 bits (bfloat16), where an exact 16-bit q uses the second
// column for nothing.  A bfloat16 cache under float32 activations takes a
// second product with the third part (X2).  INT8 keys and values are float16
// integers, exactly.
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

// truncating pack of two floats to the 16-bit type
template <bool BF>
TL_DEV int pack2(float a, float b) {
    if constexpr (BF) return (int)__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    else return __builtin_bit_cast(int, __builtin_amdgcn_cvt_pkrtz(a, b));
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

template <int HD, int DT, bool X2>
struct PagedTile {
    static constexpr bool BF = DT == DT_BF16;
    static constexpr int ES = DT == DT_I8 ? 1 : 2;       // bytes per cached value
    static constexpr int KC = HD / 32;                   // S products per 16 keys
    static constexpr int KL = HD * ES / 64;              // 16-byte loads of a key row per lane
    static constexpr int VD = HD / 16;                   // dimensions of V per lane: O products
    static constexpr int VW = VD * ES / 4;               // dwords of a V row per lane
    static constexpr int PARTS = X2 ? 2 : 1;

    // first dimension of the 8 that lane group g multiplies in S product c
    TL_DEV static int q_dim(int c, int g) { return DT == DT_I8 ? (c >> 1) * 64 + 16 * g + 8 * (c & 1) : (c * 4 + g) * 8; }
};

// Workgroup (row, KV head x block of 8 heads, split); each of its wavefronts
// takes every fourth tile of 32 keys of the split's chunk, with its own m, l and
// O, joined through LDS at the end.
template <int HD, int DT, bool X2>
__global__ __launch_bounds__(64 * kAttnWaves) void paged_attention_kernel(PagedAttnArgs a) {
    using T = PagedTile<HD, DT, X2>;
    constexpr bool BF = T::BF;
    __shared__ float s_o[kAttnWaves][8][HD + 4];
    __shared__ float s_m[kAttnWaves][8], s_l[kAttnWaves][8];
    const PagedGeom& geo = a.c.g;
    const int split = blockIdx.z, row = blockIdx.x;
    const int rep = a.n_heads / geo.n_kv;
    const int blocks = (rep + 7) >> 3;
    const int kvh = (int)blockIdx.y / blocks, h0 = ((int)blockIdx.y - kvh * blocks) * 8;
    const int heads = min(8, rep - h0);
    const int seq = a.row_seq ? a.row_seq[row] : row;
    const int pos = a.row_pos[row];
    const PagedRow kind = paged_row_kind(geo, seq, pos);
    if (kind != PAGED_ROW_OK) {
        if (kind == PAGED_ROW_FAULT && a.fault && threadIdx.x == 0) *a.fault = 1;
        return;
    }
    const int n = __builtin_amdgcn_readfirstlane(max(pos + 1, 0));
    const int64_t head0 = (int64_t)kvh * rep + h0;
    if (n == 0) {   // no keys: zeros
        if (split == 0)
            for (int i = threadIdx.x; i < heads * HD / 4; i += 64 * kAttnWaves)
                store4(a.out, (int64_t)row * a.out_stride + head0 * HD + 4 * i, a.act, v4f{0, 0, 0, 0});
        return;
    }
    const int chunk = paged_chunk(n, a.splits);
    if ((int64_t)split * chunk >= n) return;
    const int begin = split * chunk, end = (int)min((int64_t)n, (int64_t)begin + chunk);
    const int lane = lane_id(), wave = wave_id(), col = lane & 15, g = lane >> 4;
    const bool lo = col >= 8;
    const int head = col & 7;

    // the query head's parts, scaled by a power of two so that float16 holds them
    v4i qf[T::PARTS][T::KC];
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
            float part[T::PARTS][8];
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
            for (int p = 0; p < T::PARTS; p++)
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
    const unsigned lo_mask = lo ? (BF ? 0xFFFF0000u : 0xFFFFE000u) : 0u;
    const int last8 = (n - 1) & ~7;
    const char* kbase = (const char*)a.c.k;
    const char* vbase = (const char*)a.c.v;
    bool bad = false;

    for (int kb = begin + 32 * wave; kb < end; kb += 32 * kAttnWaves) {
        // key rows of S^T: row m of tile t is key kb + 8 (m / 4) + 4 t + m % 4.
        // Groups of 8 keys lie in one page; groups behind the last key read its group.
        const int kg = min(kb + 8 * (col >> 2), last8), vg = min(kb + 8 * g, last8);
        const int kp = paged_page(geo, seq, kg), vp = paged_page(geo, seq, vg);
        const char* kr = kbase + T::ES * (paged_row(geo, max(kp, 0), kvh, kg) + (col & 3) * HD) + 16 * g;
        const char* vr = vbase + T::ES * paged_row(geo, max(vp, 0), kvh, vg) + col * (T::VW * 4);
        v4i kf[2][T::KL];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < T::KL; i++) kf[t][i] = *(const v4i*)(kr + t * 4 * HD * T::ES + i * 64);
        unsigned vf[8][T::VW];
#pragma unroll
        for (int r = 0; r < 8; r++) __builtin_memcpy(vf[r], __builtin_assume_aligned(vr + r * HD * T::ES, T::VW * 4), T::VW * 4);

        v4f s[2] = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}};
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int c = 0; c < T::KC; c++) {
                v4i kk;
                if constexpr (DT == DT_I8) {
                    const unsigned w0 = (unsigned)kf[t][c >> 1][2 * (c & 1)], w1 = (unsigned)kf[t][c >> 1][2 * (c & 1) + 1];
                    kk = v4i{i8_pair_f16(__builtin_amdgcn_perm(0u, w0, 0x0C010C00u)), i8_pair_f16(__builtin_amdgcn_perm(0u, w0, 0x0C030C02u)),
                             i8_pair_f16(__builtin_amdgcn_perm(0u, w1, 0x0C010C00u)), i8_pair_f16(__builtin_amdgcn_perm(0u, w1, 0x0C030C02u))};
                } else {
                    kk = kf[t][c];
                }
#pragma unroll
                for (int p = 0; p < T::PARTS; p++) s[t] = mfma32<BF>(kk, qf[p][c], s[t]);
            }

        // lane: keys kb + 8 g + 4 t + i of its head, both parts' products added
        float x[8], mt = -__builtin_inff();
        const bool whole = kb + 32 <= n && __builtin_amdgcn_ballot_w64(vp < 0) == 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float d = s[j >> 2][j & 3];
            x[j] = (d + lane_xor<8>(d)) * cs;
        }
        if (!whole) {
            bad |= vp < 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool in = vp >= 0 && kb + 8 * g + j < n;
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
        v4i pf[T::PARTS];
        {
            float part[T::PARTS][8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float p = __builtin_amdgcn_exp2f(x[j] - off);
                l += p;
                const float r = p - __uint_as_float(__float_as_uint(p) & lo_mask);
                part[0][j] = r;
                if constexpr (X2) {
                    const float hi = __uint_as_float(__float_as_uint(p) & 0xFFFF0000u), rest = p - hi;
                    part[1][j] = lo ? 0.0f : rest - __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
                }
            }
#pragma unroll
            for (int p = 0; p < T::PARTS; p++)
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
            for (int p = 0; p < T::PARTS; p++) o[d] = mfma32<BF>(vv, pf[p], o[d]);
        }
    }
    if (a.fault && bad) *a.fault = 1;

    // both parts of a head, then the wavefronts; lane: dimensions HD/4 g + VD i + d
    l += lane_xor<16>(l);
    l += lane_xor<32>(l);
#pragma unroll
    for (int d = 0; d < T::VD; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float v = o[d][i] + lane_xor<8>(o[d][i]);
            if (!lo) s_o[wave][head][HD / 4 * g + T::VD * i + d] = v;
        }
    if (lane < 8) {
        s_m[wave][lane] = m;
        s_l[wave][lane] = l;
    }
    __syncthreads();
    const float sv = DT == DT_I8 ? a.c.vs[kvh] : 1.0f;
    for (int i = threadIdx.x; i < heads * HD / 4; i += 64 * kAttnWaves) {
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
            acc += e * *(const v4f*)&s_o[w][h][d];
        }
        acc *= sv;
        if (a.splits == 1) {
            store4(a.out, (int64_t)row * a.out_stride + (head0 + h) * HD + d, a.act, acc / ll);
        } else {
            const int64_t part = ((int64_t)row * a.n_heads + head0 + h) * a.splits + split;
            *(v4f*)(a.scratch + part * HD + d) = acc;
            if (d == 0) {
                float* ml = a.scratch + (int64_t)a.rows * a.n_heads * a.splits * HD + 2 * part;
                ml[0] = mm;
                ml[1] = ll;
            }
        }
    }
}

// the parts of one (row, head) joined: M = max m, out = sum 2^(m - M) O / sum 2^(m - M) l
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    constexpr int Q = HD / 4, W = 256 / Q;   // quads of a row; parts taken side by side
    __shared__ float s_acc[W][HD];
    __shared__ float s_l[W];
    const PagedGeom& geo = a.c.g;
    const int head = blockIdx.y, row = blockIdx.x;
    const int seq = a.row_seq ? a.row_seq[row] : row;
    const int pos = a.row_pos[row];
    if (paged_row_kind(geo, seq, pos) != PAGED_ROW_OK || pos < 0) return;
    const int parts = paged_active(pos + 1, a.splits);
    const int64_t first = ((int64_t)row * a.n_heads + head) * a.splits;
    const float* ml = a.scratch + (int64_t)a.rows * a.n_heads * a.splits * HD + 2 * first;
    const int q = threadIdx.x % Q, w = threadIdx.x / Q;
    float mm = -__builtin_inff();
    for (int i = 0; i < parts; i++) mm = fmaxf(mm, ml[2 * i]);
    const float off = mm == -__builtin_inff() ? 0.0f : mm;
    v4f acc = {0, 0, 0, 0};
    float ll = 0.0f;
    for (int i = w; i < parts; i += W) {
        const float e = __builtin_amdgcn_exp2f(ml[2 * i] - off);
        ll += e * ml[2 * i + 1];
        acc += e * *(const v4f*)(a.scratch + (first + i) * HD + 4 * q);
    }
    *(v4f*)&s_acc[w][4 * q] = acc;
    if (q == 0) s_l[w] = ll;
    __syncthreads();
    if (w != 0) return;
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
    TL_KLAUNCH(paged_append_kernel, dim3(a.rows, (units + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError();
}

int32_t paged_attention_splits(const PagedCache& c, int32_t rows, int32_t n_heads) {
    const int64_t units = (int64_t)rows * c.g.n_kv * head_blocks(n_heads, c.g.n_kv);
    const int64_t cap = ((int64_t)c.g.max_pages << c.g.page_shift);
    const int64_t most = (cap + kPagedTile - 1) / kPagedTile;
    const int64_t want = (1024 + units - 1) / std::max<int64_t>(units, 1);
    return (int32_t)std::max<int64_t>(1, std::min<int64_t>({want, most, 256}));
}

size_t paged_attention_scratch(const PagedCache& c, int32_t rows, int32_t n_heads, int32_t splits) {
    return splits <= 1 ? 0 : (size_t)rows * n_heads * splits * (c.g.head_dim + 2);
}

hipError_t launch_paged_attention(hipStream_t s, const PagedAttnArgs& a) {
    if (a.rows <= 0) return hipSuccess;
    const dim3 grid(a.rows, a.c.g.n_kv * head_blocks(a.n_heads, a.c.g.n_kv), a.splits), block(64 * kAttnWaves);
    const bool x2 = a.c.dtype == DT_BF16 && a.act != DT_BF16;
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (a.c.dtype == DT_I8) TL_KLAUNCH((paged_attention_kernel<HD, DT_I8, false>), grid, block, 0, s, a);
        else if (a.c.dtype == DT_F16) TL_KLAUNCH((paged_attention_kernel<HD, DT_F16, false>), grid, block, 0, s, a);
        else if (x2) TL_KLAUNCH((paged_attention_kernel<HD, DT_BF16, true>), grid, block, 0, s, a);
        else TL_KLAUNCH((paged_attention_kernel<HD, DT_BF16, false>), grid, block, 0, s, a);
        if (a.splits > 1) TL_KLAUNCH((paged_join_kernel<HD>), dim3(a.rows, a.n_heads), dim3(256), 0, s, a);
    };
    if (a.c.g.head_dim == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
    return hipGetLastError();
}

}  // namespace tl
