// tl_w4.hip -- projections of a few rows with 4-bit weights and group scales.
//
// y[m][n] = (residual +) sum_g s[n][g] sum_{k in g} w[n][k] x[m][k], w in -8 .. 7.
//
// The inner sums run on the INT8 matrix instructions, exactly.  A nibble becomes
// the INT8 number 16 w by a mask (and a shift for the low one).  128 columns of a row
// of x become four base-256 digits, each -128 .. 127: they are scaled by a power of two
// of their own so that their largest magnitude lies in [2^29, 2^30) and rounded to
// integers v, whose digits are the bytes of (v + 0x808080) ^ 0x808080.  So a value is
// off by at most 2^-30 of the largest of its 128 columns, whatever its type (with one
// power for a whole row, an outlier took bits from all of it: 4096 columns with one of
// 30000 times the rest lost a factor of 80 against float32); products and sums over a
// group are exact in INT32, and only the sum over groups, each times its scale, rounds,
// in float32.  The 16 columns of a product are four rows of x with four digits.
//
// What bounds it: the weights, k / 2 bytes a row, read once; of the rest the
// latency from the first load to the result.  They stream in the order of the
// lanes' registers, 1 KiB for 16 rows by 128 columns, 8 KiB in flight in each
// wavefront; the digits of up to 16 rows of x wait in LDS.  Rows of x, scales and the
// first weights are asked for together, and a block of x turns to digits as soon as it
// is there: only the sums need to know the whole row's largest magnitude (with one
// power of two for a row, and a barrier before its digits, four rows by 5632 x 2048
// took 8.5 us, now 7.9).  Queued back to back, one row by 5632 x 2048 takes 7.8 us (5.8
// in a graph), by 32000 x 2048 (group 32, float32 scales) 11.8, by 14336 x 8192 14.5
// (4.1 TB/s); 13 rows by 2048 x 5632 14.4, 16 by 32000 x 2048 20.5.  With the weights
// in the rows' own order, where a load's pieces lie k / 2 bytes apart, the second took
// 20.9.
#include <algorithm>

#include "tl_rows.h"

namespace tl {
namespace {

constexpr int kW4Ahead = 8;          // 1 KiB weight blocks in flight per wavefront
constexpr int kBadRow = INT32_MIN;   // exponent of a row with an infinity or NaN

// The digits of `cols / 4` rows of x (cols: 4, 8 or 16), in the order the products
// take them: for 64 columns of x, lane group g and column of the product 16 bytes,
// those of x's columns 32 c + 8 g + 2 i + parity at 8 c + 4 parity + i.
TL_DEV int w4_frag(int k64, int g, int col, int cols) { return ((k64 * 4 + g) * cols + col) * 16; }

// four integers (of columns k, k + 2, k + 4, k + 6) to one dword per digit
TL_DEV void digits4(int v0, int v1, int v2, int v3, unsigned d[4]) {
    const unsigned u0 = ((unsigned)v0 + 0x00808080u) ^ 0x00808080u, u1 = ((unsigned)v1 + 0x00808080u) ^ 0x00808080u;
    const unsigned u2 = ((unsigned)v2 + 0x00808080u) ^ 0x00808080u, u3 = ((unsigned)v3 + 0x00808080u) ^ 0x00808080u;
    const unsigned a = __builtin_amdgcn_perm(u1, u0, 0x05010400u), b = __builtin_amdgcn_perm(u3, u2, 0x05010400u);
    const unsigned c = __builtin_amdgcn_perm(u1, u0, 0x07030602u), e = __builtin_amdgcn_perm(u3, u2, 0x07030602u);
    d[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    d[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    d[2] = __builtin_amdgcn_perm(e, c, 0x05040100u);
    d[3] = __builtin_amdgcn_perm(e, c, 0x07060302u);
}

// Rows of x to digits by a whole workgroup: kW4Slots units of 8 columns per thread.  A
// block of 128 columns (16 adjacent threads) takes the power of two that brings its
// largest magnitude to [2^29, 2^30), so that none waits for another.
struct RowUnits {
    v4i raw[kW4Slots][2];

    // slot j: unit u0 + threadIdx.x + (j % per) * kW4Threads of row row0 + j / per, zeros
    // behind the rows and the columns
    TL_DEV void load(const W4Args& a, int row0, int rows, int per, int u0) {
        const int units = a.k >> 3;
#pragma unroll
        for (int j = 0; j < kW4Slots; j++) {
            const int r = j / per, u = u0 + threadIdx.x + (j - r * per) * kW4Threads;
            raw[j][0] = raw[j][1] = v4i{0, 0, 0, 0};
            if (r >= rows || u >= units) continue;
            const int64_t at = (row0 + r) * a.x_stride + 8 * (int64_t)u;
            if (a.act == DT_F32) {
                raw[j][0] = *(const v4i*)((const float*)a.x + at);
                raw[j][1] = *(const v4i*)((const float*)a.x + at + 4);
            } else {
                raw[j][0] = *(const v4i*)((const uint16_t*)a.x + at);
            }
        }
    }

    // digits to base, zero from column k on; bexp[4 block + row]: the blocks' powers of two;
    // most[j * kW4Waves + wave]: the largest magnitude (as bits) of the wavefront's slot j,
    // not less than what is there if `more`
    TL_DEV void digits(const W4Args& a, int rows, int per, int u0, char* base, int cols, int16_t* bexp, unsigned* most,
                       bool more) {
        const int padded = w4_blocks(a.k) * 16;
#pragma unroll
        for (int j = 0; j < kW4Slots; j++) {
            const int r = j / per, u = u0 + threadIdx.x + (j - r * per) * kW4Threads;
            if (r >= rows) break;
            v4f x[2];
#pragma unroll
            for (int h = 0; h < 2; h++)
                x[h] = a.act == DT_F32 ? __builtin_bit_cast(v4f, raw[j][h])
                                       : unpack4(v2i{raw[j][0][2 * h], raw[j][0][2 * h + 1]}, a.act);
            // magnitudes order as their bits do, infinity and NaN above the numbers
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(fabsf(x[i >> 2][i & 3])));
            m = max(m, (unsigned)dpp<kDppXor1>((int)m));
            m = max(m, (unsigned)dpp<kDppXor2>((int)m));
            m = max(m, (unsigned)dpp<kDppHalfMirror>((int)m));
            m = max(m, (unsigned)dpp<kDppRowMirror>((int)m));
            const unsigned all = max(max((unsigned)row_value((int)m, 0), (unsigned)row_value((int)m, 1)),
                                     max((unsigned)row_value((int)m, 2), (unsigned)row_value((int)m, 3)));
            const int slot = j * kW4Waves + wave_id();
            if (lane_id() == 0) most[slot] = more ? max(most[slot], all) : all;
            if (u >= padded) continue;
            const int e = fit(m);
            put(x[0], x[1], e, r, u, base, cols);
            if ((u & 15) == 0) bexp[(u >> 4) * 4 + r] = (int16_t)(e == kBadRow ? 0 : e);
        }
    }

    // the power of two that brings a largest magnitude (its bits) to [2^29, 2^30); of zeros
    // one above all others, so that a block of them counts by little
    static TL_DEV int fit(unsigned m) {
        return m >= 0x7F800000u ? kBadRow : m == 0 ? 255 : 30 - __builtin_amdgcn_frexp_expf(__uint_as_float(m));
    }

    // that of a whole row, its slots' maxima being n words
    static TL_DEV int fit_row(const unsigned* most, int n) {
        unsigned m = 0;
        for (int i = 0; i < n; i += 4) {
            const v4i v = *(const v4i*)(most + i);
            m = max(max(m, (unsigned)v[0]), max(max((unsigned)v[1], (unsigned)v[2]), (unsigned)v[3]));
        }
        return fit(m);
    }

    static TL_DEV void put(v4f x0, v4f x1, int e, int r, int u, char* base, int cols) {
        const bool bad = e == kBadRow;
        int v[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = bad ? 0 : (int)__builtin_rintf(__builtin_amdgcn_ldexpf(x0[j], e));
            v[4 + j] = bad ? 0 : (int)__builtin_rintf(__builtin_amdgcn_ldexpf(x1[j], e));
        }
        unsigned even[4], odd[4];
        digits4(v[0], v[2], v[4], v[6], even);
        digits4(v[1], v[3], v[5], v[7], odd);
        char* to = base + 8 * (u >> 2 & 1);
#pragma unroll
        for (int d = 0; d < 4; d++)
            *(v2i*)(to + w4_frag(u >> 3, u & 3, 4 * r + d, cols)) = v2i{(int)even[d], (int)odd[d]};
    }
};

__global__ __launch_bounds__(kW4Threads) void w4_digits_kernel(W4Args a) {
    __shared__ __align__(16) unsigned most[kW4Slots * kW4Waves];
    const int row = blockIdx.x, padded = w4_blocks(a.k) * 16;
    char* s = (char*)a.scratch;
    // one row at its place among its four
    char* base = s + w4_digit_off(a.m, a.k) + (row >> 2) * w4_frag_bytes(a.k, 16) + (row & 3) * 64;
    int16_t* bexp = (int16_t*)(s + w4_bexp_off(a.m) + (row >> 2) * w4_bexp_bytes(a.k)) + (row & 3);
    for (int u0 = 0; u0 < padded; u0 += kW4Slots * kW4Threads) {
        RowUnits x;
        x.load(a, row, 1, kW4Slots, u0);
        x.digits(a, 1, kW4Slots, u0, base, 16, bexp, most, u0 > 0);
    }
    __syncthreads();
    if (threadIdx.x == 0) ((int*)s)[row] = RowUnits::fit_row(most, kW4Slots * kW4Waves);
}

// What the sums of a block's digits count by: 2^-32, less what the block was scaled by
// beyond its row.  2^-22 of the result then for rows around 1, so that no partial sum
// overflows whose result does not.
TL_DEV float count_by(int row, int block) {
    return __builtin_amdgcn_ldexpf(1.0f, max(row, -1000) - block - 32);   // (a row that is not finite: any, its result is NaN)
}

struct W4Shape {
    int32_t split;       // wavefronts that share a tile of 16 weight rows: 1, 2, 4 or 8
    int32_t cols;        // columns of a product in use by the digits' layout
};

constexpr int kFirst = 4;     // fours of scales of a thread that are loaded ahead

// Workgroup (8 / split tiles of 16 weight rows, 4 CB rows of x).  LQ: log2 of the
// groups in 128 columns.  Up to four rows of x each workgroup converts to digits
// itself (COPY false); of more, it copies what w4_digits_kernel left in scratch,
// 1024 columns at a time, the next ones on their way while these are used.
template <int CB, int LQ, bool COPY>
__global__ __launch_bounds__(kW4Threads, CB < 4 ? 4 : 2) void w4_kernel(W4Args a, W4Shape sh) {
    extern __shared__ __align__(16) char lds[];
    constexpr int Q = 1 << LQ;
    const int nblk = w4_blocks(a.k), groups = nblk << LQ;
    const int lane = lane_id(), wave = wave_id(), col = lane & 15, g = lane >> 4;
    const int tiles = w4_tiles(a.n), per = kW4Waves / sh.split;
    const int part = wave % sh.split;
    const int tile = blockIdx.x * per + wave / sh.split;
    const int m0 = blockIdx.y * (4 * CB);

    // everything the workgroup starts with, on its way at once: its rows of x, the first
    // scales, the first weights
    RowUnits x;
    const int slots = w4_slots(1, a.k);   // of a row
    if constexpr (!COPY) x.load(a, m0, min(4, a.m - m0), slots, 0);
    // COPY: what the row blocks' blocks count by, from the exponents of rows and blocks, [nblk][CB] fours
    struct Exps {
        v4i row;
        v2i block;   // int16
    };
    auto block_exps = [&](int i) {
        const int b = w4_row_block(blockIdx.y, CB, i % CB, a.m), blk = min(i / CB, nblk - 1);
        return Exps{((const v4i*)a.scratch)[b], ((const v2i*)((const char*)a.scratch + w4_bexp_off(a.m) + b * w4_bexp_bytes(a.k)))[blk]};
    };
    auto counts = [&](Exps e) {
        v4f f;
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = count_by(e.row[j], (int16_t)(e.block[j >> 1] >> (16 * (j & 1))));
        return f;
    };
    Exps exps0 = {};
    if constexpr (COPY) exps0 = block_exps(threadIdx.x);

    // scales of the workgroup's tiles as float32 [tile][group][16 rows]
    float* s_scale = (float*)lds;
    const int n4 = min(per, tiles - (int)blockIdx.x * per) * groups * 4;   // fours of them
    const bool wide = a.scale_dtype == DT_F32;
    const char* sc = (const char*)a.packed + (int64_t)tiles * nblk * 1024 + (int64_t)blockIdx.x * per * groups * 16 * (wide ? 4 : 2);
    v4i first[kFirst];
#pragma unroll
    for (int j = 0; j < kFirst; j++) {
        const int i = min((int)threadIdx.x + j * kW4Threads, n4 - 1);
        if (wide) {
            first[j] = ((const v4i*)sc)[i];
        } else {
            const v2i v = ((const v2i*)sc)[i];
            first[j] = v4i{v[0], v[1], 0, 0};
        }
    }

    const char* w = (const char*)a.packed + ((int64_t)min(tile, tiles - 1) * nblk) * 1024 + lane * 16;
    v4i ring[kW4Ahead];
    auto load = [&](int i) {   // the i-th block of this wavefront
        const int blk = min(part + i * sh.split, nblk - 1);
        return __builtin_nontemporal_load((const v4i*)(w + (int64_t)blk * 1024));
    };
#pragma unroll
    for (int i = 0; i < kW4Ahead; i++) ring[i] = load(i);

    auto put_scales = [&](v4i v, int i) {
        *(v4f*)(s_scale + 4 * i) = wide ? __builtin_bit_cast(v4f, v) : unpack4(v2i{v[0], v[1]}, a.scale_dtype);
    };
    char* next = lds + (size_t)per * groups * 64;
    float* red = (float*)next;                     // [wave][16 rows][4 CB]
    next += kW4Waves * 16 * 4 * CB * 4;
    int* s_exp = (int*)next;                       // [4 CB]
    unsigned* s_most = (unsigned*)next + 16;       // [kW4Slots][wave]
    next += 192;
    float* s_by = (float*)next;                    // COPY: [nblk][CB][4]
    int16_t* s_bexp = (int16_t*)next;              // else [nblk][4]
    next += CB * nblk * 16;
    char* digits = next;
    const char* scr = (const char*)a.scratch + w4_digit_off(a.m, a.k);

    // COPY: a chunk's digits, [CB][blocks] of 2 KiB; a thread's share of the next one
    constexpr int kBlockBytes = 128 * 16, kShare = kW4Chunk * kBlockBytes / (kW4Threads * 16);
    const int64_t fcb = COPY ? kW4Chunk * kBlockBytes : 0;
    v4i share[CB][kShare];
    auto fetch = [&](int chunk) {
        const int rest = (nblk - chunk * kW4Chunk) * (kBlockBytes / 16);   // pieces of a row block from the chunk on
#pragma unroll
        for (int c = 0; c < CB; c++)
#pragma unroll
            for (int j = 0; j < kShare; j++)
                share[c][j] = ((const v4i*)(scr + w4_row_block(blockIdx.y, CB, c, a.m) * w4_frag_bytes(a.k, 16) +
                                            (int64_t)chunk * kW4Chunk * kBlockBytes))
                    [min((int)threadIdx.x + j * kW4Threads, rest - 1)];
    };
    auto put = [&](int chunk) {
#pragma unroll
        for (int c = 0; c < CB; c++)
#pragma unroll
            for (int j = 0; j < kShare; j++)
                ((v4i*)(digits + ((chunk & 1) * CB + c) * fcb))[threadIdx.x + j * kW4Threads] = share[c][j];
    };
    if constexpr (COPY) {
        if (threadIdx.x < 4 * CB) s_exp[threadIdx.x] = m0 + (int)threadIdx.x < a.m ? ((const int*)a.scratch)[m0 + threadIdx.x] : 0;
        fetch(0);
    } else {
        x.digits(a, min(4, a.m - m0), slots, 0, digits, sh.cols, s_bexp, s_most, false);
    }
#pragma unroll
    for (int j = 0; j < kFirst; j++)
        if ((int)threadIdx.x + j * kW4Threads < n4) put_scales(first[j], threadIdx.x + j * kW4Threads);
    for (int i = threadIdx.x + kFirst * kW4Threads; i < n4; i += kW4Threads)
        put_scales(wide ? ((const v4i*)sc)[i] : v4i{((const v2i*)sc)[i][0], ((const v2i*)sc)[i][1], 0, 0}, i);
    if constexpr (COPY) {
        if ((int)threadIdx.x < CB * nblk) ((v4f*)s_by)[threadIdx.x] = counts(exps0);
#pragma unroll 1
        for (int i = threadIdx.x + kW4Threads; i < CB * nblk; i += kW4Threads) ((v4f*)s_by)[i] = counts(block_exps(i));
        put(0);
    }
    __syncthreads();

    v4f acc[CB];
#pragma unroll
    for (int c = 0; c < CB; c++) acc[c] = v4f{0, 0, 0, 0};
    const int mine = (nblk - part + sh.split - 1) / sh.split;   // blocks of this wavefront
    const float* scale = s_scale + (wave / sh.split) * groups * 16 + 4 * g;
    const int frag = w4_frag(0, g, col & (sh.cols - 1), sh.cols);
    const int xrow = (col & (sh.cols - 1)) >> 2;   // this lane's row of a row block
    int rexp = 0;
    if constexpr (!COPY) {
        rexp = RowUnits::fit_row(s_most + xrow * slots * kW4Waves, slots * kW4Waves);
        if (wave == 0 && g == 0 && (col & 3) == 0) s_exp[col >> 2] = rexp;   // read behind the next barrier
    }
    const int f64 = 4 * sh.cols * 16;              // bytes of 64 columns' digits

    auto block = [&](v4i q, int blk, const char* base) {
        const v4i lo = (q << 4) & (int)0xF0F0F0F0, hi = q & (int)0xF0F0F0F0;
        v4f sc[Q];
#pragma unroll
        for (int j = 0; j < Q; j++) sc[j] = *(const v4f*)(scale + ((blk << LQ) + j) * 16);
        int at = blk * CB * 4;
        asm volatile("" : "+s"(at));   // (or every step of the loop holds an address of its own, 30 registers)
#pragma unroll
        for (int c = 0; c < CB; c++) {
            const char* f = base + c * fcb + frag;
            const float by = COPY ? s_by[at + c * 4 + xrow] : count_by(rexp, s_bexp[at + xrow]);
            v4i t = {0, 0, 0, 0};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const v4i b = *(const v4i*)(f + h * f64);
                const v4i aw = {lo[2 * h], hi[2 * h], lo[2 * h + 1], hi[2 * h + 1]};
                if constexpr (LQ < 2) {
                    if (LQ == 1) t = v4i{0, 0, 0, 0};
                    t = __builtin_amdgcn_mfma_i32_16x16x64_i8(aw, b, t, 0, 0, 0);
                    if (LQ == 1 || h == 1)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            acc[c][i] = __builtin_fmaf((float)t[i] * by, sc[LQ == 1 ? h : 0][i], acc[c][i]);
                } else {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const long aa = __builtin_bit_cast(long, v2i{aw[2 * e], aw[2 * e + 1]});
                        const long bb = __builtin_bit_cast(long, v2i{b[2 * e], b[2 * e + 1]});
                        const v4i u = __builtin_amdgcn_mfma_i32_16x16x32_i8(aa, bb, v4i{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            acc[c][i] = __builtin_fmaf((float)u[i] * by, sc[(2 * h + e) & (Q - 1)][i], acc[c][i]);
                    }
                }
            }
        }
    };
    if constexpr (COPY) {
        // every wavefront goes through all chunks, as they meet at each
        const int chunks = (nblk + kW4Chunk - 1) / kW4Chunk, each = kW4Chunk / sh.split;   // its blocks in a chunk
        fetch(min(1, chunks - 1));
        for (int i0 = 0; i0 < chunks * each; i0 += kW4Ahead) {
#pragma unroll
            for (int s = 0; s < kW4Ahead; s++) {
                const int i = i0 + s;
                if (i >= chunks * each) break;
                const int ch = i / each;
                if (i > 0 && (s & (each - 1)) == 0) {
                    // (the buffer's last readers were done before the chunk in between began)
                    put(ch);
                    __syncthreads();
                    if (ch + 1 < chunks) fetch(ch + 1);
                }
                if (i < mine) {
                    const int blk = part + i * sh.split;
                    const v4i q = ring[s];
                    ring[s] = load(i + kW4Ahead);
                    block(q, blk, digits + (ch & 1) * CB * fcb + (blk - ch * kW4Chunk) * kBlockBytes);
                }
            }
        }
    } else {
        for (int i0 = 0; i0 < mine; i0 += kW4Ahead) {
#pragma unroll
            for (int s = 0; s < kW4Ahead; s++) {
                if (i0 + s >= mine) break;
                const v4i q = ring[s];
                ring[s] = load(i0 + s + kW4Ahead);   // (behind the last block: the last again)
                const int blk = part + (i0 + s) * sh.split;
                block(q, blk, digits + (int64_t)blk * 2 * f64);
            }
        }
    }

    // a row of x: its digits' columns, each 256^(digit - 3) of the result; then the wavefronts
    // of a tile
    const float place = __builtin_amdgcn_ldexpf(1.0f, 8 * (col & 3) - 24);
#pragma unroll
    for (int c = 0; c < CB; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v = acc[c][i] * place;
            v += lane_xor<1>(v);
            v += lane_xor<2>(v);
            if ((col & 3) == 0) red[(wave * 16 + 4 * g + i) * (4 * CB) + 4 * c + (col >> 2)] = v;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < per * 16 * 4 * CB; i += kW4Threads) {
        const int r = i & 15, m = (i >> 4) % (4 * CB), t = (i >> 4) / (4 * CB);
        const int64_t nn = ((int64_t)blockIdx.x * per + t) * 16 + r;
        if (nn >= a.n || m0 + m >= a.m) continue;
        float v = 0.0f;
        for (int p = 0; p < sh.split; p++) v += red[((t * sh.split + p) * 16 + r) * (4 * CB) + m];
        const int e = s_exp[m];
        v = e == kBadRow ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(v, 52 - e);   // 2^e x, 2^4 w, 2^-56
        if (a.residual) v += load1(a.residual, (m0 + m) * a.res_stride + nn, a.act);
        store1(a.y, (m0 + m) * a.y_stride + nn, a.act, v);
    }
}

// one 16-byte piece of the packed weights, or four scales, per thread
__global__ __launch_bounds__(256) void pack_w4_kernel(const uint8_t* q, const void* scales, int dt, int group, int n, int k,
                                                      char* packed) {
    const int nblk = w4_blocks(k), tiles = w4_tiles(n), groups = w4_groups(k, group), ng = k / group;
    const int64_t pieces = (int64_t)tiles * nblk * 64, quads = (int64_t)tiles * groups * 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces + quads; i += (int64_t)gridDim.x * 256) {
        if (i < pieces) {
            const int lane = (int)(i & 63), blk = (int)((i >> 6) % nblk);
            const int64_t row = (i >> 6) / nblk * 16 + (lane & 15);
            v4i v = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int byte = blk * 64 + 16 * j + 4 * (lane >> 4);
                if (row < n && byte < k / 2) v[j] = *(const int*)(q + row * (k / 2) + byte);
            }
            *(v4i*)(packed + i * 16) = v;
        } else {
            const int64_t s = i - pieces;
            const int64_t row = s / (groups * 4) * 16 + 4 * (s & 3);
            const int gr = (int)((s >> 2) % groups);
            v4f v = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (row + j < n && gr < ng) v[j] = load1(scales, (row + j) * ng + gr, dt);
            store4(packed + pieces * 16, s * 4, dt, v);
        }
    }
}

// ---------------------------------------------------------------------------
// quantizer: per group s = max|w| / 7 rounded to the scales' type (1 where that
// is zero), w4 = clip(rne(w / s), -8, 7).  A thread takes 8 columns.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void quantize_w4_kernel(const float* w, int64_t total8, int k, int group, int dt,
                                                          uint8_t* q, void* scales) {
    for (int64_t u0 = (int64_t)blockIdx.x * 256; u0 < total8; u0 += (int64_t)gridDim.x * 256) {
        const int64_t u = u0 + threadIdx.x;
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
        if (u >= total8) continue;
        *(unsigned*)(q + (at >> 1)) = out;
        if (at % group == 0) store1(scales, at / group, dt, s);
    }
}

int log2_groups(int32_t group) { return group == 128 ? 0 : group == 64 ? 1 : 2; }

}  // namespace

bool w4_supported(int32_t k, int32_t group) {
    return (group == 32 || group == 64 || group == 128) && k > 0 && k % group == 0 && k / group <= kW4MaxGroups;
}

int64_t w4_packed_bytes(int32_t n, int32_t k, int32_t group, int32_t scale_dtype) {
    return (int64_t)w4_tiles(n) * (w4_blocks(k) * 1024ll + w4_groups(k, group) * 16ll * (scale_dtype == DT_F32 ? 4 : 2));
}

hipError_t launch_linear_w4(hipStream_t s, const W4Args& a) {
    if (a.m <= 0 || a.n <= 0) return hipSuccess;
    const W4Plan p = w4_plan(a.m, a.n, a.k, a.group);
    if (!p.convert) TL_KLAUNCH(w4_digits_kernel, dim3(a.m), dim3(kW4Threads), 0, s, a);
    const W4Shape sh{p.split, p.cols};
    const dim3 grid(p.grid_x, p.grid_y), block(kW4Threads);
    const size_t lds = p.lds;
    auto go = [&](auto cbt, auto copyt) {
        constexpr int CB = decltype(cbt)::value;
        constexpr bool COPY = decltype(copyt)::value;
        switch (log2_groups(a.group)) {
            case 0: TL_KLAUNCH((w4_kernel<CB, 0, COPY>), grid, block, lds, s, a, sh); break;
            case 1: TL_KLAUNCH((w4_kernel<CB, 1, COPY>), grid, block, lds, s, a, sh); break;
            default: TL_KLAUNCH((w4_kernel<CB, 2, COPY>), grid, block, lds, s, a, sh); break;
        }
    };
    using std::integral_constant;
    if (p.convert) go(integral_constant<int, 1>{}, std::false_type{});
    else if (p.cb == 1) go(integral_constant<int, 1>{}, std::true_type{});
    else if (p.cb == 2) go(integral_constant<int, 2>{}, std::true_type{});
    else go(integral_constant<int, 4>{}, std::true_type{});
    return hipGetLastError();
}

hipError_t launch_pack_w4(hipStream_t s, const uint8_t* q, const void* scales, int32_t scale_dtype, int32_t group,
                          int32_t n, int32_t k, void* packed) {
    const int64_t work = (int64_t)w4_tiles(n) * (w4_blocks(k) * 64ll + w4_groups(k, group) * 4ll);
    TL_KLAUNCH(pack_w4_kernel, dim3((unsigned)std::min<int64_t>(8192, (work + 255) / 256)), dim3(256), 0, s, q, scales,
               scale_dtype, group, n, k, (char*)packed);
    return hipGetLastError();
}

hipError_t launch_quantize_w4(hipStream_t s, const float* w, int32_t rows, int32_t k, int32_t group, int32_t scale_dtype,
                              uint8_t* q, void* scales) {
    const int64_t total8 = (int64_t)rows * k / 8;
    if (total8 <= 0) return hipSuccess;
    TL_KLAUNCH(quantize_w4_kernel, dim3(w4_quantize_grid(total8)), dim3(256), 0, s, w, total8, k, group, scale_dtype, q,
               scales);
    return hipGetLastError();
}

template <int CB, bool COPY>
static hipError_t init_w4() {
    hipError_t e = hipSuccess;
    for (const void* f : {(const void*)w4_kernel<CB, 0, COPY>, (const void*)w4_kernel<CB, 1, COPY>, (const void*)w4_kernel<CB, 2, COPY>})
        if (e == hipSuccess) e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, kW4Lds);
    return e;
}

hipError_t init_w4_kernels() {
    hipError_t e;
    if ((e = init_w4<1, false>()) || (e = init_w4<1, true>()) || (e = init_w4<2, true>()) || (e = init_w4<4, true>())) return e;
    return hipSuccess;
}

}  // namespace tl
