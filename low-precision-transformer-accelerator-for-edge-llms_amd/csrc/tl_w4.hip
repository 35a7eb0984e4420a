// tl_w4.hip -- projections of a few rows with 4-bit weights and group scales.
//
// y[m][n] = (residual +) sum_g s[n][g] sum_{k in g} w[n][k] x[m][k], w in -8 .. 7.
//
// The inner sums run on v_mfma_i32_16x16x64_i8, exactly: a nibble becomes the
// INT8 number 16 w by a mask (and a shift for the low one), and a row of x
// becomes four base-256 digits, each -128 .. 127.  The row is scaled by a power
// of two so that its largest magnitude lies in [2^29, 2^30) and rounded to an
// integer v; the digits are the bytes of (v + 0x808080) ^ 0x808080.  A value is
// off by at most 2^-30 of its row's largest, whatever its type; products and
// sums of 128 are exact in INT32, and only the sum over groups (each times its
// scale) rounds, in float32.
//
// A matrix product has 16 columns, a row of x takes four of them (its digits),
// times the groups in the product's 128 weights: with groups of 64 or 32 each
// group has columns of its own that are zero in the others' places.
#include <algorithm>

#include "tl_rows.h"

namespace tl {
namespace {

constexpr int kW4Waves = 8;
constexpr int kW4MaxGroups = 1024;   // group scales of a row held in LDS
constexpr int kBadRow = INT32_MIN;   // exponent of a row with an infinity or NaN
constexpr int kZeros = 128;          // bytes of zeros the unused columns read

__host__ __device__ inline int w4_blocks(int k) { return 2 * ((k + 255) / 256); }   // 128-weight blocks, in pairs
// bytes of one digit of a row, shifted 16 per digit so that columns differ in LDS bank
__host__ __device__ inline int w4_digit_stride(int k) { return w4_blocks(k) * 128 + 16; }

// four integers (of columns k, k + 2, k + 4, k + 6) to one dword per digit
TL_DEV void digits4(const int v[4], unsigned d[4]) {
    unsigned u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = ((unsigned)v[i] + 0x00808080u) ^ 0x00808080u;
    const unsigned a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
    const unsigned c = __builtin_amdgcn_perm(u[1], u[0], 0x07030602u), e = __builtin_amdgcn_perm(u[3], u[2], 0x07030602u);
    d[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    d[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    d[2] = __builtin_amdgcn_perm(e, c, 0x05040100u);
    d[3] = __builtin_amdgcn_perm(e, c, 0x07060302u);
}

// The digits of one row of x at base[digit][block][column parity][lane group]
// [16]: byte j of lane group g in block b is column 128 b + 32 g + 2 j + parity,
// as the low and high nibbles of a lane's 16 weight bytes come.  Columns from k
// on are zero.  Returns the power of two the row was scaled by (kBadRow: not
// finite).  The whole workgroup takes part; red: a word per wavefront.
template <typename P>
TL_DEV int row_digits(const W4Args& a, int64_t row, P base, unsigned* red) {
    const int nt = blockDim.x;
    const int64_t at = row * a.x_stride;
    unsigned mx = 0;
    for (int i = threadIdx.x * 4; i < a.k; i += nt * 4) {
        const v4f v = load4(a.x, at + i, a.act);
#pragma unroll
        for (int j = 0; j < 4; j++) mx = max(mx, __float_as_uint(fabsf(v[j])));
    }
    // magnitudes order as their bits do, infinity and NaN above the numbers
#pragma unroll
    for (int o = 32; o; o >>= 1) mx = max(mx, (unsigned)__shfl_xor((int)mx, o));
    __syncthreads();
    if (lane_id() == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    for (int i = 0; i < nt >> 6; i++) mx = max(mx, red[i]);
    const bool bad = mx >= 0x7F800000u;
    const int e = bad || mx == 0 ? 0 : 30 - __builtin_amdgcn_frexp_expf(__uint_as_float(mx));
    const int ds = w4_digit_stride(a.k);
    for (int i = threadIdx.x * 8; i < w4_blocks(a.k) * 128; i += nt * 8) {
        v4f x0 = {0, 0, 0, 0}, x1 = {0, 0, 0, 0};
        if (i < a.k && !bad) {   // k is a multiple of 32
            x0 = load4(a.x, at + i, a.act);
            x1 = load4(a.x, at + i + 4, a.act);
        }
        int v[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            v[j][0] = (int)__builtin_rintf(__builtin_amdgcn_ldexpf(x0[j], e));
            v[j][1] = (int)__builtin_rintf(__builtin_amdgcn_ldexpf(x0[2 + j], e));
            v[j][2] = (int)__builtin_rintf(__builtin_amdgcn_ldexpf(x1[j], e));
            v[j][3] = (int)__builtin_rintf(__builtin_amdgcn_ldexpf(x1[2 + j], e));
        }
        const int to = (i >> 7) * 128 + ((i >> 5) & 3) * 16 + ((i >> 3) & 3) * 4;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            unsigned d[4];
            digits4(v[j], d);
#pragma unroll
            for (int c = 0; c < 4; c++) *(unsigned*)(base + c * ds + to + 64 * j) = d[c];
        }
    }
    return bad ? kBadRow : e;
}

// scratch of a call: zeros, the rows' exponents, the rows' digits
__host__ __device__ inline size_t w4_exp_off() { return kZeros; }
__host__ __device__ inline size_t w4_digit_off(int m) { return kZeros + ((size_t)m * 4 + 15) / 16 * 16; }

__global__ __launch_bounds__(512) void w4_digits_kernel(W4Args a) {
    __shared__ unsigned red[8];
    const int row = blockIdx.x;
    char* s = (char*)a.scratch;
    if (row == 0 && threadIdx.x < kZeros / 4) ((unsigned*)s)[threadIdx.x] = 0u;
    const int e = row_digits(a, row, s + w4_digit_off(a.m) + (size_t)row * 4 * w4_digit_stride(a.k), red);
    if (threadIdx.x == 0) ((int*)(s + w4_exp_off()))[row] = e;
}

// Workgroup (16 weight rows, tile of x rows): its wavefronts share out the pairs
// of 128-weight blocks of the rows; CB column blocks of 16.
template <int CB>
__global__ __launch_bounds__(64 * kW4Waves) void w4_kernel(W4Args a, int lq) {
    extern __shared__ __align__(16) char lds[];
    const int ng = a.k / a.group, nblk = w4_blocks(a.k);
    const int q_n = 1 << lq;                           // groups in a block
    const int cols = 4 << lq;                          // columns of one row of x
    const int mt = (CB * 16) >> (2 + lq);              // rows of x in a tile
    const int m0 = blockIdx.y * mt, n0 = blockIdx.x * 16;
    const int lane = lane_id(), wave = wave_id(), col = lane & 15, g = lane >> 4;

    // the first weights, on their way while the scales are laid out
    const int64_t row_bytes = a.k >> 1;
    const uint8_t* wrow = a.q + (int64_t)min(n0 + col, a.n - 1) * row_bytes;
    auto load = [&](int blk) {
        const int64_t at = blk * 64 + g * 16;
        return at < row_bytes ? __builtin_nontemporal_load((const v4i*)(wrow + at)) : v4i{0, 0, 0, 0};
    };
    const int pairs = nblk >> 1;
    v4i next[2] = {};
    if (wave < pairs) {
        next[0] = load(2 * wave);
        next[1] = load(2 * wave + 1);
    }

    // scales as float32, [group][16 rows], zeros behind the last group
    float* s_w = (float*)lds;
    for (int i = threadIdx.x; i < 16 * nblk * q_n; i += 64 * kW4Waves) {
        const int r = i / (nblk * q_n), gr = i - r * (nblk * q_n);
        s_w[gr * 16 + r] = gr < ng ? load1(a.scales, (int64_t)min(n0 + r, a.n - 1) * ng + gr, a.scale_dtype) : 0.0f;
    }
    float* red = s_w + 16 * nblk * q_n;                // [wave][16 rows][mt]

    // where this lane reads each column block's digits: its column's row and digit,
    // or zeros where its column is another group's or past the last row
    const char* scr = (const char*)a.scratch;
    const int ds = w4_digit_stride(a.k);
    const char* b_at[CB];
    int b_step[CB];
#pragma unroll
    for (int c = 0; c < CB; c++) {
        const int cc = c * 16 + col, m = m0 + (cc >> (2 + lq)), d = (cc >> lq) & 3;
        const bool mine = m < a.m && (g >> (2 - lq)) == (cc & (q_n - 1));
        b_at[c] = mine ? scr + w4_digit_off(a.m) + ((size_t)m * 4 + d) * ds + g * 16 : scr;
        b_step[c] = mine ? 128 : 0;
    }
    v4f acc[CB];
#pragma unroll
    for (int c = 0; c < CB; c++) acc[c] = v4f{0, 0, 0, 0};
    __syncthreads();

    for (int p = wave; p < pairs; p += kW4Waves) {
        const v4i cur[2] = {next[0], next[1]};
        if (p + kW4Waves < pairs) {
            next[0] = load(2 * (p + kW4Waves));
            next[1] = load(2 * (p + kW4Waves) + 1);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int blk = 2 * p + h;
            const v4i lo = (cur[h] << 4) & (int)0xF0F0F0F0, hi = cur[h] & (int)0xF0F0F0F0;
            const v4f sc = *(const v4f*)(s_w + ((blk << lq) + (col & (q_n - 1))) * 16 + 4 * g);
#pragma unroll
            for (int c = 0; c < CB; c++) {
                const char* b = b_at[c] + (int64_t)blk * b_step[c];
                v4i t = {0, 0, 0, 0};
                t = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo, *(const v4i*)b, t, 0, 0, 0);
                t = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi, *(const v4i*)(b + 64), t, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) acc[c][i] = __builtin_fmaf((float)t[i], sc[i], acc[c][i]);
            }
        }
    }

    // columns of a row of x: its digits, times 256^digit, and its groups
#pragma unroll
    for (int c = 0; c < CB; c++) {
        const float w = __builtin_amdgcn_ldexpf(1.0f, 8 * ((col >> lq) & 3));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v = acc[c][i] * w;
            for (int o = 1; o < cols; o <<= 1) v += lane_xor_rt(v, o);
            if ((col & (cols - 1)) == 0) red[(wave * 16 + 4 * g + i) * mt + ((c * 16 + col) >> (2 + lq))] = v;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * mt; i += 64 * kW4Waves) {
        const int r = i & 15, m = i >> 4;
        if (n0 + r >= a.n || m0 + m >= a.m) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kW4Waves; w++) v += red[(w * 16 + r) * mt + m];
        const int e = ((const int*)(scr + w4_exp_off()))[m0 + m];
        v = e == kBadRow ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(v, -e - 4);   // the weights came as 16 w
        if (a.residual) v += load1(a.residual, (int64_t)(m0 + m) * a.res_stride + n0 + r, a.act);
        store1(a.y, (int64_t)(m0 + m) * a.y_stride + n0 + r, a.act, v);
    }
}

// ---------------------------------------------------------------------------
// quantizer: per group s = max|w| / 7 rounded to the scales' type (1 where that
// is zero), w4 = clip(rne(w / s), -8, 7).  A thread takes 8 columns.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void quantize_w4_kernel(const float* w, int64_t total8, int k, int group, int dt,
                                                          uint8_t* q, void* scales) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t at = min(u, total8 - 1) * 8;         // idle lanes repeat the last unit
    const v4f x0 = *(const v4f*)(w + at), x1 = *(const v4f*)(w + at + 4);
    float mx = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) mx = fmaxf(mx, fmaxf(fabsf(x0[j]), fabsf(x1[j])));
    mx = fmaxf(mx, lane_xor<1>(mx));
    mx = fmaxf(mx, lane_xor<2>(mx));
    if (group >= 64) mx = fmaxf(mx, lane_xor<4>(mx));
    if (group >= 128) mx = fmaxf(mx, lane_xor<8>(mx));
    float s = __fdiv_rn(mx, 7.0f);
    if (dt == DT_BF16) s = bf16_bits(to_bf16(s));
    if (dt == DT_F16) s = f16_bits(to_f16(fminf(s, 65504.0f)));
    const bool zero = s == 0.0f;
    if (zero) s = 1.0f;
    unsigned out = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float v = zero ? 0.0f : __builtin_rintf(__fdiv_rn(j < 4 ? x0[j & 3] : x1[j & 3], s));
        v = v > 7.0f ? 7.0f : v;
        v = v >= -8.0f ? v : -8.0f;
        out |= ((unsigned)(int)v & 15u) << (4 * j);
    }
    if (u >= total8) return;
    *(unsigned*)(q + (at >> 1)) = out;
    if (at % group == 0) store1(scales, at / group, dt, s);
}

}  // namespace

bool w4_supported(int32_t k, int32_t group) {
    return (group == 32 || group == 64 || group == 128) && k > 0 && k % group == 0 && k / group <= kW4MaxGroups;
}

size_t w4_scratch(int32_t m, int32_t n, int32_t k, int32_t group) {
    (void)n;
    (void)group;
    return w4_digit_off(m) + (size_t)m * 4 * w4_digit_stride(k);
}

static size_t w4_lds(int32_t k, int lq, int mt) {
    return ((size_t)16 * (w4_blocks(k) << lq) + (size_t)kW4Waves * 16 * mt) * sizeof(float);
}

hipError_t launch_linear_w4(hipStream_t s, const W4Args& a) {
    if (a.m <= 0 || a.n <= 0) return hipSuccess;
    TL_KLAUNCH(w4_digits_kernel, dim3(a.m), dim3(512), 0, s, a);
    const int lq = a.group == 128 ? 0 : a.group == 64 ? 1 : 2;
    auto go = [&](auto cbt) {
        constexpr int CB = decltype(cbt)::value;
        const int mt = (CB * 16) >> (2 + lq);
        const dim3 grid((a.n + 15) / 16, (a.m + mt - 1) / mt);
        TL_KLAUNCH((w4_kernel<CB>), grid, dim3(64 * kW4Waves), w4_lds(a.k, lq, mt), s, a, lq);
    };
    const int cb = ((a.m << (2 + lq)) + 15) / 16;
    if (cb <= 1) go(std::integral_constant<int, 1>{});
    else if (cb <= 2) go(std::integral_constant<int, 2>{});
    else if (cb <= 4) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
    return hipGetLastError();
}

hipError_t launch_quantize_w4(hipStream_t s, const float* w, int32_t rows, int32_t k, int32_t group, int32_t scale_dtype,
                              uint8_t* q, void* scales) {
    const int64_t total8 = (int64_t)rows * k / 8;
    if (total8 <= 0) return hipSuccess;
    TL_KLAUNCH(quantize_w4_kernel, dim3((unsigned)((total8 + 255) / 256)), dim3(256), 0, s, w, total8, k, group, scale_dtype, q,
               scales);
    return hipGetLastError();
}

hipError_t init_w4_kernels() {
    hipError_t e = hipSuccess;
    auto big = [&](const void* f) {
        if (e == hipSuccess) e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    };
    big((const void*)w4_kernel<1>);
    big((const void*)w4_kernel<2>);
    big((const void*)w4_kernel<4>);
    big((const void*)w4_kernel<8>);
    return e;
}

}  // namespace tl
