// tl_paged.hip -- the paged KV cache: append with rotation, and the attention of
// one query row per token over it.
#include <algorithm>

#include "tl_attn.h"

namespace tl {
namespace {

// ---------------------------------------------------------------------------
// append: q and k of each row rotated at its position (TL:69-80, the steps of
// tl_rope: two products and their sum, each rounded to float32), k and v written
// to the row's place in the cache (INT8: clip(rne(x / s), +-127) with a float32
// division, as tl_qkv_append), q written out in the activations' type.
// A workgroup takes 256 units of one row: a unit is four rotated pairs (d ..
// d + 3 and their partners half a head on), or eight values of v.  Nothing is
// read twice from memory; the row's cos and sin are shared by its heads through
// the cache.  With gains, q and k of each head are normed first: f = 1 / sqrt(mean x^2 +
// eps) in 64 bits, rounded once (or, where float32 holds it as no normal number, not
// rounded), so that neither the order of the sum nor a square root's
// last bit shows in an INT8 row; then (x f) gain, each product rounded to float32.  A head's
// pairs lie in 8 or 16 neighbouring lanes, which add up their squares with DPP moves.  What bounds it: from one row to some hundreds the chain of loads and
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

// sum over the 8 or 16 lanes that hold a head's rotated pairs, in every one of them
TL_DEV double head_sum(double v, int quads) {
    auto add = [&](auto ctrl) {
        constexpr int CTRL = decltype(ctrl)::value;
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const unsigned lo = (unsigned)dpp<CTRL>((int)(unsigned)u), hi = (unsigned)dpp<CTRL>((int)(unsigned)(u >> 32));
        v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    add(std::integral_constant<int, kDppXor1>{});
    add(std::integral_constant<int, kDppXor2>{});
    add(std::integral_constant<int, kDppHalfMirror>{});
    if (quads == 16) add(std::integral_constant<int, kDppRowMirror>{});
    return v;
}

template <int ACT, bool NORM>
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
    v4f x1 = load4(a.qkv, at, ACT), x2 = load4(a.qkv, at + (rotate ? half : 4), ACT);
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
        if constexpr (NORM) {
            const float* gain = head < a.n_heads ? a.q_gain : a.k_gain;
            if (gain) {
                const v4f g1 = *(const v4f*)(gain + d), g2 = *(const v4f*)(gain + d + half);
                double sum = 0.0;
#pragma unroll
                for (int j = 0; j < 4; j++) sum += (double)x1[j] * x1[j] + (double)x2[j] * x2[j];
                const double wide = 1.0 / __builtin_sqrt(head_sum(sum, quads) / hd + a.eps);
                const float f = (float)wide;
                if (f >= 0x1p-126f && f < __builtin_inff()) {
                    x1 *= f;
                    x2 *= f;
                } else {   // a factor that float32 does not hold whole: heads near either end of its range
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        x1[j] = (float)(x1[j] * wide);
                        x2[j] = (float)(x2[j] * wide);
                    }
                }
                x1 *= g1;
                x2 *= g2;
            }
        }
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
template <int HD, int DT, bool X2>
__global__ __launch_bounds__(kAttnThreads, 2) void paged_attention_kernel(PagedAttnArgs a) {
    __shared__ AttnShared<HD, DT, X2> sh;
    attention_run<HD, DT, X2, false>(a, blockIdx.x, gridDim.x, sh);
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
        const LaneRows l = lane_rows<false>(a, all);
        share = paged_share((int32_t)all * hbs, workgroups);
        tiles = (int)tiles_at<false>(a, pos);
        const int kvh = head / rep, hb = kvh * blocks + ((head - kvh * rep) >> 3);
        unit = __builtin_amdgcn_readlane((int)(l.upto - l.tiles), row) * hbs + hb * tiles;
    } else {
        const int w = blockIdx.x + 1;
        RowScan first;
        const int32_t total = __builtin_amdgcn_readfirstlane(count_tiles<false>(a, s_scan, first));
        share = paged_share(total * hbs, workgroups);
        const int32_t at = share.start(w);
        if (at >= total * hbs || at == share.start(w - 1)) return;
        int32_t before;
        find_row<false>(a, s_scan, (unsigned)at / (unsigned)hbs, first, row, before);
        tiles = (int)tiles_at<false>(a, a.row_pos[row]);
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
    auto go = [&](auto norm) {
        constexpr bool NORM = decltype(norm)::value;
        if (a.act == DT_F32) TL_KLAUNCH((paged_append_kernel<DT_F32, NORM>), grid, block, 0, s, a);
        else if (a.act == DT_BF16) TL_KLAUNCH((paged_append_kernel<DT_BF16, NORM>), grid, block, 0, s, a);
        else TL_KLAUNCH((paged_append_kernel<DT_F16, NORM>), grid, block, 0, s, a);
    };
    if (a.q_gain || a.k_gain) go(std::true_type{});
    else go(std::false_type{});
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
    if (args.prefix.len > 0) return launch_shared_attention(s, args);
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
