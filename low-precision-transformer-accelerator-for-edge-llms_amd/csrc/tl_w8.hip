// tl_w8.hip -- projections with 8-bit weights and 8-bit activations: INT8 matrix
// products with a scale for each token and each channel, alone or as the gate and up
// projections of a feed-forward block with their product.
//
// s_m = max |x_m| / 127 (1 where that is 0), q_m = clip(rne(x_m / s_m), +-127), each step
// in float32; y[m][n] = (sum_k q[m][k] w[n][k]) s_n s_m (+ residual), the sum exact in
// INT32, its conversion and the two products float32; the scales' powers of two come last,
// so that nothing on the way leaves the range that the result is in.  Gated: y = silu(gate) up of two
// such results, silu(g) = g / (1 + e^-g).
//
// Weights lie in blocks of 16 rows and 64 columns, 1 KiB in the order of a wavefront's
// registers for v_mfma_i32_16x16x64_i8 (lane l: row l % 16, columns 16 (l / 16) .. + 15),
// and so do the quantized rows of x.  Weights are the rows of a product and tokens its
// columns, so that a lane's four results are neighbours in a row of y.
#include <algorithm>

#include "tl_rows.h"

namespace tl {
namespace {

// Rows may start anywhere their type may: wide loads and stores need no more than that of
// the address.
typedef int v4i_any __attribute__((ext_vector_type(4), aligned(2)));
typedef int v2i_any __attribute__((ext_vector_type(2), aligned(2)));

// Eight columns of a row of x, as they lie in memory; zeros behind column k.
struct Unit {
    v4i raw[2];

    TL_DEV void load(const W8Args& a, int64_t row, int u) {
        raw[0] = raw[1] = v4i{0, 0, 0, 0};
        const int left = a.k - 8 * u;
        if (left <= 0) return;
        const int64_t at = row * a.x_stride + 8 * (int64_t)u;
        if (left >= 8) {
            if (a.act == DT_F32) {
                raw[0] = *(const v4i_any*)((const float*)a.x + at);
                raw[1] = *(const v4i_any*)((const float*)a.x + at + 4);
            } else {
                raw[0] = *(const v4i_any*)((const uint16_t*)a.x + at);
            }
            return;
        }
        if (a.act == DT_F32) {
            const int* p = (const int*)a.x + at;
#pragma unroll
            for (int i = 0; i < 8; i++) raw[i >> 2][i & 3] = i < left ? p[i] : 0;
        } else {
            const uint16_t* p = (const uint16_t*)a.x + at;
#pragma unroll
            for (int i = 0; i < 8; i++) raw[0][i >> 1] |= (i < left ? (int)p[i] : 0) << (16 * (i & 1));
        }
    }
    TL_DEV v4f get(int h, int act) const {
        return act == DT_F32 ? __builtin_bit_cast(v4f, raw[h]) : unpack4(v2i{raw[0][2 * h], raw[0][2 * h + 1]}, act);
    }
    // the largest magnitude, as bits: they order as magnitudes do, infinity and NaN above
    TL_DEV unsigned most(int act) const {
        unsigned m = 0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const v4f v = get(h, act);
#pragma unroll
            for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(fabsf(v[i])));
        }
        return m;
    }
    TL_DEV v2i quantized(int act, const RnDiv& d) const {
        const v4f lo = get(0, act), hi = get(1, act);
        const float4 a = {lo[0], lo[1], lo[2], lo[3]}, b = {hi[0], hi[1], hi[2], hi[3]};
        if (d.fast) return v2i{(int)quant4<true>(a, d), (int)quant4<true>(b, d)};
        return v2i{(int)quant4<false>(a, d), (int)quant4<false>(b, d)};
    }
};

// A row's scale from its largest magnitude's bits.  A row with an infinity or NaN has the
// scale NaN (its results are NaN) and quantizes to zeros.
TL_DEV bool row_finite(unsigned most) { return most < 0x7F800000u; }
TL_DEV float row_scale(unsigned most) {
    if (!row_finite(most)) return __builtin_nanf("");
    const float s = __fdiv_rn(__uint_as_float(most), 127.0f);
    return s == 0.0f ? 1.0f : s;
}

TL_DEV unsigned wave_max_u32(unsigned m) {
    m = max(m, (unsigned)dpp<kDppXor1>((int)m));
    m = max(m, (unsigned)dpp<kDppXor2>((int)m));
    m = max(m, (unsigned)dpp<kDppHalfMirror>((int)m));
    m = max(m, (unsigned)dpp<kDppRowMirror>((int)m));
    return max(max((unsigned)row_value((int)m, 0), (unsigned)row_value((int)m, 1)),
               max((unsigned)row_value((int)m, 2), (unsigned)row_value((int)m, 3)));
}

TL_DEV const float* w8_scales(const W8Args& a) {
    return (const float*)((const char*)a.packed + (int64_t)w8_tiles(a.n, a.glu) * w8_blocks(a.k) * 1024);
}
TL_DEV float* w8_row_scales(const W8Args& a) { return (float*)a.scratch; }
TL_DEV char* w8_rows_at(const W8Args& a) { return (char*)a.scratch + w8_rows_off(a.m); }

// silu(g) u.  Below -80 silu is taken as -0 (its magnitude is below 2e-33).
TL_DEV float glu(float g, float u) {
    if (g < -80.0f) return -0.0f * u;
    const float t = tl_expf_nonpos(-fabsf(g));
    return __fdiv_rn(g >= 0.0f ? g : g * t, 1.0f + t) * u;
}

// four neighbours of a row of the residual from column n on, zeros behind the last column
TL_DEV v4f w8_residual(const W8Args& a, int64_t m, int n) {
    const int64_t at = m * a.res_stride + n;
    if (n + 4 <= a.n) {
        if (a.act == DT_F32) return __builtin_bit_cast(v4f, (v4i)*(const v4i_any*)((const float*)a.residual + at));
        return unpack4(*(const v2i_any*)((const uint16_t*)a.residual + at), a.act);
    }
    v4f v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < a.n) v[i] = load1(a.residual, at + i, a.act);
    return v;
}
// and of y
TL_DEV void w8_store(const W8Args& a, int64_t m, int n, v4f v) {
    const int64_t at = m * a.y_stride + n;
    if (n + 4 <= a.n) {
        if (a.act == DT_F32) {
            *(v4i_any*)((float*)a.y + at) = __builtin_bit_cast(v4i, v);
            return;
        }
        v2i w;
        store4(&w, 0, a.act, v);
        *(v2i_any*)((uint16_t*)a.y + at) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < a.n) store1(a.y, at + i, a.act, v[i]);
}
TL_DEV void w8_put(const W8Args& a, int64_t m, int n, v4f v) {
    if (a.residual) v += w8_residual(a, m, n);
    w8_store(a, m, n, v);
}

// results of 4 rows of a weight tile (from row 4 g of it) for token m: sums to y
TL_DEV v4f w8_scaled(v4i sum, v4f sw, float sx) {
    v4f v;
#pragma unroll
    for (int i = 0; i < 4; i++)
        v[i] = __builtin_amdgcn_ldexpf((float)sum[i] * __builtin_amdgcn_frexp_mantf(sw[i]) * __builtin_amdgcn_frexp_mantf(sx),
                                       __builtin_amdgcn_frexp_expf(sw[i]) + __builtin_amdgcn_frexp_expf(sx));
    return v;
}
TL_DEV v4f w8_glu(v4i gate, v4i up, v4f sg, v4f su, float sx) {
    const v4f g = w8_scaled(gate, sg, sx), u = w8_scaled(up, su, sx);
    v4f v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = glu(g[i], u[i]);
    return v;
}

// Steps 0 .. count - 1 of which the first AHEAD have been fetched into sets 0 .. AHEAD - 1:
// multiply(set, step), fetch(set, step).  No step is fetched behind the last one, and in the
// loop none under a condition, which would have the compiler wait for all that are on their way.
template <int AHEAD, typename Multiply, typename Fetch>
TL_DEV void in_flight(int count, Multiply multiply, Fetch fetch) {
    int i0 = 0;
    for (; i0 + 2 * AHEAD <= count; i0 += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            multiply(j, i0 + j);
            fetch(j, i0 + j + AHEAD);
        }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; j++) {
        if (i0 + j < count) multiply(j, i0 + j);
        if (j + 1 < AHEAD && i0 + j + AHEAD < count) fetch(j, i0 + j + AHEAD);
    }
#pragma unroll
    for (int j = 0; j + 1 < AHEAD; j++)
        if (i0 + j + AHEAD < count) multiply(j, i0 + j + AHEAD);
}

// ---------------------------------------------------------------------------
// Rows of x to INT8 blocks and scales in scratch, `waves` wavefronts to a row.
// ---------------------------------------------------------------------------
template <int ACT>
__global__ __launch_bounds__(kW8Threads, 8) void w8_quantize_kernel(W8Args a, int waves) {
    a.act = ACT;
    __shared__ unsigned s_most[kW8Waves];
    const int wave = wave_id(), part = wave % waves;
    const int row = blockIdx.x * (kW8Waves / waves) + wave / waves;
    const int blocks = w8_blocks(a.k), units = blocks * 8, step = 64 * waves;
    const bool in = row < a.m;
    Unit x[kW8Keep];
    unsigned most = 0;
    if (in) {
#pragma unroll
        for (int j = 0; j < kW8Keep; j++) x[j].load(a, row, part * 64 + lane_id() + j * step);
#pragma unroll
        for (int j = 0; j < kW8Keep; j++) most = max(most, x[j].most(a.act));
        for (int u = part * 64 + lane_id() + kW8Keep * step; u < units; u += step) {
            Unit y;
            y.load(a, row, u);
            most = max(most, y.most(a.act));
        }
    }
    most = wave_max_u32(most);
    if (waves > 1) {
        if (lane_id() == 0) s_most[wave] = most;
        __syncthreads();
        most = 0;
        for (int w = 0; w < waves; w++) most = max(most, s_most[wave - part + w]);
    }
    if (!in) return;
    const float s = row_scale(most);
    const bool finite = row_finite(most);
    const RnDiv d = rn_div_prep(finite ? s : 1.0f);
    if (part == 0 && lane_id() == 0) w8_row_scales(a)[row] = s;
    char* to = w8_rows_at(a) + (int64_t)(row >> 4) * blocks * 1024 + (row & 15) * 16;
    auto put = [&](const Unit& y, int u) {
        if (u < units)
            *(v2i*)(to + (int64_t)(u >> 3) * 1024 + (u >> 1 & 3) * 256 + (u & 1) * 8) = finite ? y.quantized(a.act, d) : v2i{0, 0};
    };
#pragma unroll
    for (int j = 0; j < kW8Keep; j++) put(x[j], part * 64 + lane_id() + j * step);
    for (int u = part * 64 + lane_id() + kW8Keep * step; u < units; u += step) {
        Unit y;
        y.load(a, row, u);
        put(y, u);
    }
}

// ---------------------------------------------------------------------------
// Up to four rows whose columns its registers hold: every workgroup quantizes them itself,
// into LDS.  Rows, first weights, scales and residual are asked for together; what bounds
// it is that chain (load, maximum, quotients, products, sums: one row by 2048 x 5632 7.1 us in a
// graph, by 5632 x 2048 6.2, the gated pair 8.2) and then the weights (two sets in turn, 14336 x
// 4096: 11.2 us, 5.2 TB/s; the pair 20.3, 5.8 TB/s).
// ---------------------------------------------------------------------------
constexpr int kRowAhead = 8;   // weight blocks in flight per wavefront

template <bool GLU>
__global__ __launch_bounds__(kW8Threads, 4) void w8_row_kernel(W8Args a, int split) {
    constexpr int S = GLU ? 2 : 1, AHEAD = kRowAhead / S;
    extern __shared__ __align__(16) char lds[];   // x [block][16 columns][row][16], then partial sums
    __shared__ unsigned s_most[4][kW8Waves];
    const int lane = lane_id(), wave = wave_id(), col = lane & 15, g = lane >> 4;
    const int blocks = w8_blocks(a.k), units = blocks * 8, m = a.m;
    const int per = kW8Waves / split, part = wave % split;
    const int tiles = (a.n + 15) >> 4;
    const int tile = blockIdx.x * per + wave / split;
    const int slots = (units + kW8Threads - 1) / kW8Threads;   // of a row

    Unit x[kW8Slots];
#pragma unroll
    for (int j = 0; j < kW8Slots; j++) {
        const int r = j / slots;
        if (r < m) x[j].load(a, r, (int)threadIdx.x + (j - r * slots) * kW8Threads);
    }
    // this wavefront's weights: blocks part, part + split, ...
    const int count = tile < tiles ? (blocks - part + split - 1) / split : 0;
    const char* w[S];
#pragma unroll
    for (int s = 0; s < S; s++)
        w[s] = (const char*)a.packed + ((int64_t)(min(tile, tiles - 1) * S + s) * blocks + min(part, blocks - 1)) * 1024 + lane * 16;
    const int last = max(count - 1, 0);
    v4i wf[AHEAD][S];
#pragma unroll
    for (int j = 0; j < AHEAD; j++)
#pragma unroll
        for (int s = 0; s < S; s++) wf[j][s] = __builtin_nontemporal_load((const v4i*)(w[s] + (int64_t)min(j, last) * split * 1024));

    // what this thread finishes: four columns of y of a token
    static_assert(kW8Waves * 4 * 4 <= kW8Threads, "one item to a thread");
    const int fr = (int)threadIdx.x / (per * 4), fq = (int)threadIdx.x - fr * (per * 4), ft = blockIdx.x * per + (fq >> 2);
    const bool finishes = fr < m && ft < tiles;
    v4f sw[S], res = {0, 0, 0, 0};
    if (finishes) {
#pragma unroll
        for (int s = 0; s < S; s++) sw[s] = *(const v4f*)(w8_scales(a) + (ft * S + s) * 16 + 4 * (fq & 3));
        if (a.residual) res = w8_residual(a, fr, ft * 16 + 4 * (fq & 3));
    }

    unsigned most[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kW8Slots; j++) {
        const int r = j / slots;
        if (r >= m) break;
        const unsigned v = x[j].most(a.act);
#pragma unroll
        for (int i = 0; i < 4; i++) most[i] = i == r ? max(most[i], v) : most[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i >= m) break;
        const unsigned v = wave_max_u32(most[i]);
        if (lane == 0) s_most[i][wave] = v;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i >= m) break;
        most[i] = 0;
#pragma unroll
        for (int v = 0; v < kW8Waves; v++) most[i] = max(most[i], s_most[i][v]);
    }
#pragma unroll
    for (int j = 0; j < kW8Slots; j++) {
        const int r = j / slots, u = (int)threadIdx.x + (j - r * slots) * kW8Threads;
        if (r >= m) break;
        unsigned mr = most[0];
#pragma unroll
        for (int i = 1; i < 4; i++) mr = i == r ? most[i] : mr;
        mr = (unsigned)__builtin_amdgcn_readfirstlane((int)mr);
        const bool finite = row_finite(mr);
        const RnDiv d = rn_div_prep(finite ? row_scale(mr) : 1.0f);
        if (u < units) *(v2i*)(lds + ((u >> 1) * m + r) * 16 + (u & 1) * 8) = finite ? x[j].quantized(a.act, d) : v2i{0, 0};
    }
    __syncthreads();

    v4i acc[S];
#pragma unroll
    for (int s = 0; s < S; s++) acc[s] = v4i{0, 0, 0, 0};
    const char* xl = lds + (g * m + min(col, m - 1)) * 16;
    auto multiply = [&](int j, int i) {
        const v4i xf = *(const v4i*)(xl + (int64_t)(part + i * split) * 64 * m);
#pragma unroll
        for (int s = 0; s < S; s++) acc[s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j][s], xf, acc[s], 0, 0, 0);
    };
    auto fetch = [&](int j, int i) {
#pragma unroll
        for (int s = 0; s < S; s++) wf[j][s] = __builtin_nontemporal_load((const v4i*)(w[s] + (int64_t)i * split * 1024));
    };
    in_flight<AHEAD>(count, multiply, fetch);
    // parts of a tile meet in LDS: [wave][s][4 g][16 columns] fours
    char* red = lds + (int64_t)blocks * 64 * m;
#pragma unroll
    for (int s = 0; s < S; s++) *(v4i*)(red + (wave * S + s) * 1024 + lane * 16) = acc[s];
    __syncthreads();
    if (!finishes) return;
    v4i sum[S];
#pragma unroll
    for (int s = 0; s < S; s++) {
        sum[s] = v4i{0, 0, 0, 0};
        for (int p = 0; p < split; p++)
            sum[s] += *(const v4i*)(red + (((fq >> 2) * split + p) * S + s) * 1024 + ((fq & 3) * 16 + fr) * 16);
    }
    unsigned mr = most[0];
#pragma unroll
    for (int j = 1; j < 4; j++) mr = j == fr ? most[j] : mr;
    const float sx = row_scale(mr);
    v4f v;
    if constexpr (GLU) v = w8_glu(sum[0], sum[1], sw[0], sw[1], sx);
    else v = w8_scaled(sum[0], sw[0], sx);
    if (a.residual) v += res;
    w8_store(a, fr, ft * 16 + 4 * (fq & 3), v);
}

// Sums of NB tiles of 16 weight rows and 16 MB tokens in LDS, [MB][NB][lane] fours as a
// product leaves them, to y.  Neighbouring threads take neighbouring fours of a row.
template <int NB, int MB, bool GLU>
TL_DEV void w8_finish(const W8Args& a, const char* sums, int tile0, int m0, int threads) {
    constexpr int Q = (GLU ? NB / 2 : NB) * 4;   // fours of a row
    const int tiles = w8_tiles(a.n, a.glu);
    const float* scales = w8_scales(a);
    for (int i = threadIdx.x; i < Q * 16 * MB; i += threads) {
        const int r = i / Q, q = i - r * Q, at = q >> 2, g = q & 3;
        const int m = m0 + r;
        const int t = tile0 + (GLU ? 2 * at : at);
        if (m >= a.m || t >= tiles) continue;
        const float sx = w8_row_scales(a)[m];
        const char* s = sums + (((r >> 4) * NB + (GLU ? 2 * at : at)) * 64 + g * 16 + (r & 15)) * 16;
        const float* sw = scales + t * 16 + 4 * g;
        const int n = (GLU ? t >> 1 : t) * 16 + 4 * g;
        if constexpr (GLU)
            w8_put(a, m, n, w8_glu(*(const v4i*)s, *(const v4i*)(s + 1024), *(const v4f*)sw, *(const v4f*)(sw + 16), sx));
        else
            w8_put(a, m, n, w8_scaled(*(const v4i*)s, *(const v4f*)sw, sx));
    }
}

// ---------------------------------------------------------------------------
// Rows in scratch, few of them: a workgroup has NT tiles of 16 weight rows and MT of 16
// tokens, its wavefronts every eighth block of 64 columns, operands straight into
// registers, sums added in LDS (integers, so in any order).
// ---------------------------------------------------------------------------
template <int NT, int MT, bool GLU>
__global__ __launch_bounds__(kW8Threads, NT * MT > 8 ? 2 : 4) void w8_split_kernel(W8Args a) {
    constexpr int AHEAD = 4;
    __shared__ __align__(16) int sums[NT * MT * 256];
    const int lane = lane_id(), wave = wave_id();
    const int blocks = w8_blocks(a.k), tiles = w8_tiles(a.n, a.glu), mbs = (a.m + 15) >> 4;
    const int tile0 = blockIdx.x * NT, mb0 = blockIdx.y * MT;
    const char* w[NT];
    const char* x[MT];
#pragma unroll
    for (int i = 0; i < NT; i++) w[i] = (const char*)a.packed + (int64_t)min(tile0 + i, tiles - 1) * blocks * 1024 + lane * 16;
#pragma unroll
    for (int j = 0; j < MT; j++) x[j] = w8_rows_at(a) + (int64_t)min(mb0 + j, mbs - 1) * blocks * 1024 + lane * 16;
    const int count = wave < blocks ? (blocks - wave + kW8Waves - 1) / kW8Waves : 0;
    const int last = max(count - 1, 0);
    v4i wf[AHEAD][NT], xf[AHEAD][MT];
    auto fetch = [&](int s, int i) {
        const int64_t at = (int64_t)min(wave + min(i, last) * kW8Waves, blocks - 1) * 1024;
#pragma unroll
        for (int j = 0; j < NT; j++) wf[s][j] = *(const v4i*)(w[j] + at);
#pragma unroll
        for (int j = 0; j < MT; j++) xf[s][j] = *(const v4i*)(x[j] + at);
    };
#pragma unroll
    for (int s = 0; s < AHEAD; s++) fetch(s, s);
    for (int i = threadIdx.x; i < NT * MT * 256; i += kW8Threads) sums[i] = 0;
    v4i acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = v4i{0, 0, 0, 0};
    __syncthreads();
    in_flight<AHEAD>(
        count,
        [&](int s, int) {
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[s][i], xf[s][j], acc[i][j], 0, 0, 0);
        },
        fetch);
    if (count > 0) {
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int j = 0; j < MT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) atomicAdd(&sums[((j * NT + i) * 64 + lane) * 4 + e], acc[i][j][e]);
    }
    __syncthreads();
    w8_finish<NT, MT, GLU>(a, (const char*)sums, tile0, mb0 * 16, kW8Threads);
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup has a tile of WN TN x WM TM blocks; wavefront (wn, wm) multiplies TN
// x TM of them.  Both operands come into LDS by global -> LDS loads, a block of 64 columns
// (a stage) at a time, kStages - 1 stages ahead in a ring.  Stage s + 1's operands are read
// from LDS to registers while stage s is multiplied.  The ring's buffers are arrays of
// their own, so that the compiler sees that a read does not wait for the loads into the
// others, and the loop goes once around the ring.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(1))) const char W8Global;
typedef __attribute__((address_space(3))) void W8Lds;
constexpr int kStages = 4;

// At most N of the wavefront's loads left, or all of its LDS reads done.  By the builtin,
// which the compiler counts with: it adds no wait of its own for what this one covers.
template <int N>
TL_DEV void wait_loads() {
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);
}
TL_DEV void wait_reads() { __builtin_amdgcn_s_waitcnt(0xC07F); }
TL_DEV void meet() { asm volatile("s_barrier" ::: "memory"); }

template <int WN, int WM, int TN, int TM, bool GLU>
__global__ __launch_bounds__(64 * WN * WM, 1) void w8_tile_kernel(W8Args a, W8Grid grid) {
    constexpr int NB = WN * TN, MB = WM * TM, WAVES = WN * WM;
    constexpr int PW = (NB + MB + WAVES - 1) / WAVES, FR = PW * WAVES;   // blocks of a stage (NB + MB in use), a wavefront's
    constexpr int ROW = TN * 64 + 16;              // bytes of a token's sums, on their way to y
    static_assert((16 * ROW + TM * 64) * ((WAVES + kStages - 1) / kStages) <= FR * 1024, "sums and scales fit the ring");
    __shared__ __align__(16) char ring0[FR * 1024], ring1[FR * 1024], ring2[FR * 1024], ring3[FR * 1024];
    const int lane = lane_id(), wave = wave_id(), wn = wave % WN, wm = wave / WN;
    const int blocks = w8_blocks(a.k), tiles = w8_tiles(a.n, a.glu), mbs = (a.m + 15) >> 4;
    int tn, tm;
    grid.tile(blockIdx.x, tn, tm);
    const int tile0 = tn * NB, mb0 = tm * MB;
    constexpr int SL = (TM * 16 + 63) / 64;        // scales of this wavefront's tokens, in each lane
    float my_scale[SL];
#pragma unroll
    for (int i = 0; i < SL; i++) my_scale[i] = w8_row_scales(a)[min((mb0 + wm * TM) * 16 + 64 * i + lane, a.m - 1)];

    const char* src[PW];
#pragma unroll
    for (int j = 0; j < PW; j++) {
        const int b = min(wave * PW + j, NB + MB - 1);
        src[j] = (b < NB ? (const char*)a.packed + (int64_t)min(tile0 + b, tiles - 1) * blocks * 1024
                         : w8_rows_at(a) + (int64_t)min(mb0 + b - NB, mbs - 1) * blocks * 1024) + lane * 16;
    }
    auto bring = [&](char* ring) {
#pragma unroll
        for (int j = 0; j < PW; j++) {
            __builtin_amdgcn_global_load_lds((W8Global*)src[j], (W8Lds*)(ring + (wave * PW + j) * 1024), 16, 0, 0);
            src[j] += 1024;
        }
    };
    v4i wf[2][TN], xf[2][TM];
    auto read = [&](int set, const char* ring) {
#pragma unroll
        for (int i = 0; i < TN; i++) wf[set][i] = *(const v4i*)(ring + (wn * TN + i) * 1024 + lane * 16);
#pragma unroll
        for (int j = 0; j < TM; j++) xf[set][j] = *(const v4i*)(ring + (NB + wm * TM + j) * 1024 + lane * 16);
    };
    v4i acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) acc[i][j] = v4i{0, 0, 0, 0};
    auto multiply = [&](int set) {
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < TM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[set][i], xf[set][j], acc[i][j], 0, 0, 0);
    };
    // Stage s, whose operands are in registers: stage s + 1 has arrived when at most the loads
    // of s + 2 and s + 3 are left; behind the barrier it is there for every wavefront, and
    // every wavefront has stage s in registers, whose buffer takes s + 4.
    auto stage = [&](int set, char* here, const char* next) {
        wait_loads<2 * PW>();
        wait_reads();
        meet();
        __builtin_amdgcn_sched_barrier(0);
        read(set ^ 1, next);
        bring(here);
        multiply(set);
        // LDS takes 8 cycles or more for a read and 8 wavefronts ask at once: the reads are
        // spread between the products, or these would wait until all are taken
        constexpr int READS = TN + TM, EACH = TN * TM / READS;
#pragma unroll
        for (int i = 0; i < READS; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if (i < PW) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, TN * TM - EACH * READS, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // one of the last stages, `left` of them and it left
    auto late = [&](int left, int set, char* here, const char* next) {
        if (left <= 0) return;
        if (left > 1) {
            if (left > 3) wait_loads<2 * PW>();
            else if (left > 2) wait_loads<PW>();
            else wait_loads<0>();
            wait_reads();
            meet();
            if (left > 4) bring(here);
            read(set ^ 1, next);
        }
        multiply(set);
    };
    bring(ring0);
    bring(ring1);   // (blocks is even)
    if (blocks > 2) {
        bring(ring2);
        bring(ring3);
        wait_loads<3 * PW>();
    } else {
        wait_loads<PW>();
    }
    meet();
    read(0, ring0);
    int left = blocks;
    for (; left >= 2 * kStages; left -= kStages) {
        stage(0, ring0, ring1);
        stage(1, ring1, ring2);
        stage(0, ring2, ring3);
        stage(1, ring3, ring0);
    }
    late(left, 0, ring0, ring1);
    late(left - 1, 1, ring1, ring2);
    late(left - 2, 0, ring2, ring3);
    late(left - 3, 1, ring3, ring0);
    late(left - 4, 0, ring0, ring1);
    late(left - 5, 1, ring1, ring2);
    // sums of 16 tokens at a time through this wavefront's part of the ring, a token's side by
    // side, so that its results are written together
    __syncthreads();
    char* mine = (wave % kStages == 0 ? ring0 : wave % kStages == 1 ? ring1 : wave % kStages == 2 ? ring2 : ring3) + wave / kStages * (16 * ROW + TM * 64);
    constexpr int Q = (GLU ? TN / 2 : TN) * 4, STEP = 64 / Q;   // fours of a token; tokens of a pass
    const int q = lane % Q, t = tile0 + wn * TN + (q >> 2) * (GLU ? 2 : 1);
    const float* scales = w8_scales(a) + min(t, tiles - 1 - GLU) * 16 + 4 * (q & 3);
    const v4f sw = *(const v4f*)scales, su = *(const v4f*)(scales + (GLU ? 16 : 0));
    const int n = (GLU ? t >> 1 : t) * 16 + 4 * (q & 3);
    float* row_scales = (float*)(mine + 16 * ROW);
#pragma unroll
    for (int i = 0; i < SL; i++)
        if (64 * i + lane < TM * 16) row_scales[64 * i + lane] = my_scale[i];
#pragma unroll
    for (int j = 0; j < TM; j++) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < TN; i++) *(v4i*)(mine + (lane & 15) * ROW + i * 64 + (lane >> 4) * 16) = acc[i][j];
        __builtin_amdgcn_wave_barrier();
        const int m0 = (mb0 + wm * TM + j) * 16;
#pragma unroll 2
        for (int r = lane < Q * STEP ? lane / Q : 16; r < 16; r += STEP) {   // (7 tiles: lanes 56 on would write again)
            if (m0 + r >= a.m || t >= tiles) continue;
            const float sx = row_scales[j * 16 + r];
            const char* from = mine + r * ROW + (q >> 2) * (GLU ? 128 : 64) + (q & 3) * 16;
            if constexpr (GLU) w8_put(a, m0 + r, n, w8_glu(*(const v4i*)from, *(const v4i*)(from + 64), sw, su, sx));
            else w8_put(a, m0 + r, n, w8_scaled(*(const v4i*)from, sw, sx));
        }
    }
}

// q [n][k] (and q2) into blocks, scales behind them; tiles of q and q2 take turns
__global__ __launch_bounds__(256) void pack_w8_kernel(const int8_t* q, const float* scales, const int8_t* q2, const float* scales2,
                                                     int n, int k, char* packed) {
    const int two = q2 ? 2 : 1, blocks = w8_blocks(k), tiles = w8_tiles(n, two == 2);
    const int64_t pieces = (int64_t)tiles * blocks * 64, work = pieces + (int64_t)tiles * 16;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < work; i += (int64_t)gridDim.x * 256) {
        if (i >= pieces) {
            const int64_t r = i - pieces;
            const int64_t tile = r >> 4, row = (two == 2 ? tile >> 1 : tile) * 16 + (r & 15);
            ((float*)(packed + pieces * 16))[r] = row < n ? (two == 2 && (tile & 1) ? scales2 : scales)[row] : 0.0f;
            continue;
        }
        const int lane = (int)(i & 63);
        const int64_t b = i >> 6, tile = b / blocks;
        const int c = (int)(b - tile * blocks) * 64 + 16 * (lane >> 4);
        const int64_t row = (two == 2 ? tile >> 1 : tile) * 16 + (lane & 15);
        const int8_t* from = two == 2 && (tile & 1) ? q2 : q;
        typedef int v4i_bytes __attribute__((ext_vector_type(4), aligned(1)));
        v4i v = {0, 0, 0, 0};
        if (row < n && c + 16 <= k) {
            v = *(const v4i_bytes*)(from + row * k + c);
        } else if (row < n) {
            for (int j = 0; j < 16; j++)
                if (c + j < k) v[j >> 2] |= (int)((unsigned)(uint8_t)from[row * k + c + j] << (8 * (j & 3)));
        }
        *(v4i*)(packed + i * 16) = v;
    }
}

}  // namespace

hipError_t launch_linear_w8(hipStream_t s, const W8Args& a) {
    if (a.m <= 0 || a.n <= 0) return hipSuccess;
    const W8Plan p = w8_plan(a.m, a.n, a.k, a.glu);
    if (p.kind == W8_ROW) {
        const dim3 grid(p.grid_x), block(kW8Threads);
        if (a.glu) TL_KLAUNCH((w8_row_kernel<true>), grid, block, p.lds, s, a, p.split);
        else TL_KLAUNCH((w8_row_kernel<false>), grid, block, p.lds, s, a, p.split);
        return hipGetLastError();
    }
    const int per = kW8Waves / p.quant_waves;
    const dim3 rows((a.m + per - 1) / per), threads(kW8Threads);
    if (a.act == DT_F32) TL_KLAUNCH((w8_quantize_kernel<DT_F32>), rows, threads, 0, s, a, p.quant_waves);
    else if (a.act == DT_BF16) TL_KLAUNCH((w8_quantize_kernel<DT_BF16>), rows, threads, 0, s, a, p.quant_waves);
    else TL_KLAUNCH((w8_quantize_kernel<DT_F16>), rows, threads, 0, s, a, p.quant_waves);
    const dim3 grid(p.grid_x, p.grid_y), block(kW8Threads);
    using std::integral_constant;
    if (p.kind == W8_SPLIT) {
        auto go = [&](auto nt, auto mt) {
            constexpr int NT = decltype(nt)::value, MT = decltype(mt)::value;
            if (a.glu) TL_KLAUNCH((w8_split_kernel<NT, MT, true>), grid, block, 0, s, a);
            else TL_KLAUNCH((w8_split_kernel<NT, MT, false>), grid, block, 0, s, a);
        };
        if (p.mt == 1) go(integral_constant<int, 2>{}, integral_constant<int, 1>{});
        else if (p.mt == 2) go(integral_constant<int, 2>{}, integral_constant<int, 2>{});
        else go(integral_constant<int, 4>{}, integral_constant<int, 4>{});
        return hipGetLastError();
    }
    auto tile = [&](auto wn, auto wm, auto tn, auto tm) {
        constexpr int WN = decltype(wn)::value, WM = decltype(wm)::value, TN = decltype(tn)::value, TM = decltype(tm)::value;
        if constexpr (TN % 2 == 0) {
            if (a.glu) {
                TL_KLAUNCH((w8_tile_kernel<WN, WM, TN, TM, true>), grid, dim3(64 * WN * WM), 0, s, a, p.tiles);
                return;
            }
        }
        TL_KLAUNCH((w8_tile_kernel<WN, WM, TN, TM, false>), grid, dim3(64 * WN * WM), 0, s, a, p.tiles);
    };
    integral_constant<int, 2> two;
    integral_constant<int, 4> four;
    switch (p.shape) {
        case W8_8x8: tile(two, two, four, four); break;
        case W8_14x16: tile(two, four, integral_constant<int, 7>{}, four); break;
        case W8_16x14: tile(four, two, four, integral_constant<int, 7>{}); break;
        default: tile(two, four, integral_constant<int, 8>{}, four); break;
    }
    return hipGetLastError();
}

hipError_t launch_pack_w8(hipStream_t s, const int8_t* q, const float* scales, const int8_t* q2, const float* scales2,
                          int32_t n, int32_t k, void* packed) {
    const int64_t work = (int64_t)w8_tiles(n, q2 != nullptr) * (w8_blocks(k) * 64ll + 16);
    TL_KLAUNCH(pack_w8_kernel, dim3((unsigned)std::min<int64_t>(8192, (work + 255) / 256)), dim3(256), 0, s, q, scales, q2,
               scales2, n, k, (char*)packed);
    return hipGetLastError();
}

}  // namespace tl
