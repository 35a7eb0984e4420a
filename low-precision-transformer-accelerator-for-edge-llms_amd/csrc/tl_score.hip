// tl_score.hip -- log probability of a given token, entropy and the most probable
// alternatives of each row of logits, in one pass over the logits.
//
// With m = max x, S = sum e^(x - m), T = sum (x - m) e^(x - m):
//   log p_i = x_i - m - ln S,   H = ln S - T / S.
// A workgroup takes 8192 logits of a row into registers (32 per thread), leaves
// its m, S, T (base 2) and its largest `top` logits; a second kernel joins the
// parts of a row.  A row of one part is finished by its own workgroup.
//
// Alternatives are ordered by logit, equal ones by index: 64-bit keys (the
// order-preserving bits of the logit above, the index's complement below), so
// the order is total.  A workgroup does not sort: the top-th largest of the
// maxima of its 64 sets of 128 logits is a lower bound of the top-th largest
// logit, and the few logits above it are ranked against each other.
#include <algorithm>

#include "tl_rows.h"

namespace tl {
namespace {

constexpr int kThreads = 256;
constexpr int kTiles = 4;                          // 8 adjacent logits per thread and tile
constexpr int kPart = kThreads * 8 * kTiles;       // logits per workgroup
constexpr int kList = 1024;                        // candidates ranked at once
constexpr float kLn2 = 0.693147180559945309417f;
constexpr float kLog2e = 1.44269504088896340736f;

TL_DEV unsigned order_bits(float v) {              // greater logits, greater bits; never 0
    if (v == 0.0f) v = 0.0f;                       // -0 and +0 are equal
    const unsigned u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Part {
    float m, s, t, pad;   // s, t relative to m, in base 2: s = sum 2^y, t = sum y 2^y, y = (x - m) log2 e
};

struct Shared {
    float set_max[64];
    float red[8];
    int count;
    int wave_count[4];
    unsigned long long list[kList];
    unsigned long long best[kMaxTop];
};

// list[0 .. n) (distinct keys, 0: none) ranked; the largest `top` to best[] in
// order.  A key's rank stops counting at `top`.
TL_DEV void rank_list(Shared& sh, int n, int top) {
    for (int i = threadIdx.x; i < top; i += kThreads) sh.best[i] = 0ull;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned long long k = sh.list[i];
        if (k == 0ull) continue;
        int r = 0;
        for (int j = 0; j < n && r < top; j++) r += sh.list[j] > k;
        if (r < top) sh.best[r] = k;
    }
    __syncthreads();
}

// what a row gives, from its m, S, T and its best keys
TL_DEV void finish_row(const LogprobsArgs& a, int64_t row, const Part& p, const unsigned long long* best) {
    const float ls = __log2f(p.s);
    if (threadIdx.x == 0) {
        const int t = a.targets[row];
        float lp = 0.0f;
        if (t >= a.vocab) {
            lp = __builtin_nanf("");
            if (a.fault) *a.fault = 1;
        } else if (t >= 0) {
            lp = (load1(a.logits, row * a.stride + t, a.dtype) - p.m) - ls * kLn2;
        }
        a.logprob[row] = lp;
        if (a.entropy) a.entropy[row] = (ls - p.t / p.s) * kLn2;
    }
    for (int i = threadIdx.x; i < a.top; i += kThreads) {
        const unsigned long long k = best[i];
        a.top_ids[row * a.top + i] = k ? key_index(k) : -1;
        a.top_logprobs[row * a.top + i] = k ? (key_logit(k) - p.m) - ls * kLn2 : __builtin_nanf("");
    }
}

// a row may start up to 7 places into its first unit
int64_t parts_of(int32_t vocab) { return ((int64_t)vocab + 7 + kPart - 1) / kPart; }

template <int DT>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobsArgs a, int parts) {
    __shared__ Shared sh;
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    const int part = blockIdx.y;
    const int64_t row = blockIdx.x;
    const char* base = (const char*)a.logits + row * a.stride * ES;
    // units of 8 start at multiples of 16 bytes: the row's first logit is at place
    // `skew` of unit 0
    const int skew = (int)((uintptr_t)base / ES & (16 / ES - 1));
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int64_t first = (int64_t)part * kPart + tid * 8 - skew;   // this thread's first index
    if (tid == 0) sh.count = 0;

    float x[kTiles][8];
#pragma unroll
    for (int t = 0; t < kTiles; t++) {
        const int64_t i = first + t * (kThreads * 8);
        if (i >= 0 && i + 8 <= a.vocab) {
            if constexpr (DT == DT_F32) {
                const v4f p = __builtin_nontemporal_load((const v4f*)(base + i * ES));
                const v4f q = __builtin_nontemporal_load((const v4f*)(base + i * ES + 16));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[t][j] = p[j];
                    x[t][4 + j] = q[j];
                }
            } else {
                const v4i w = __builtin_nontemporal_load((const v4i*)(base + i * ES));
                const v4f p = unpack4(v2i{w[0], w[1]}, DT), q = unpack4(v2i{w[2], w[3]}, DT);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[t][j] = p[j];
                    x[t][4 + j] = q[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[t][j] = i + j >= 0 && i + j < a.vocab ? load1(base, i + j, DT) : -__builtin_inff();
        }
    }

    // maximum of the workgroup, and of each set of 4 threads
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < kTiles; t++)
#pragma unroll
        for (int j = 0; j < 8; j++) mx = fmaxf(mx, x[t][j]);
    mx = fmaxf(mx, lane_xor<1>(mx));
    mx = fmaxf(mx, lane_xor<2>(mx));
    if ((lane & 3) == 0) sh.set_max[wave * 16 + (lane >> 2)] = mx;
    __syncthreads();
    const float set = fmaxf(sh.set_max[lane], -__builtin_inff());   // a set of NaN has no logit to offer
    const float m = wave_max_f32(set);

    // sums relative to the workgroup's maximum; a logit of minus infinity adds nothing
    float s = 0.0f, tt = 0.0f;
    const float off = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int t = 0; t < kTiles; t++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float y = (x[t][j] - off) * kLog2e;
            const float e = __builtin_amdgcn_exp2f(y);
            s += e;
            tt = __builtin_fmaf(fmaxf(y, -1e30f), e, tt);
        }
    s = wave_butterfly_sum(s);
    tt = wave_butterfly_sum(tt);
    if (lane == 0) {
        sh.red[wave] = s;
        sh.red[4 + wave] = tt;
    }

    if (a.top > 0) {
        // a bound no greater than the top-th largest logit: the greatest number of 16
        // leading order bits that at least `top` set maxima reach
        const unsigned key = order_bits(set);
        unsigned bound = 0;
#pragma unroll
        for (int b = 31; b >= 16; b--) {
            const unsigned c = bound | (1u << b);
            if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= c)) >= a.top) bound = c;
        }
        // ... as a logit (bound's lower bits are zero: for a negative one, the lowest of its class)
        const float low = bound == 0 ? -__builtin_inff() : __uint_as_float(bound & 0x80000000u ? bound & 0x7FFFFFFFu : ~bound);
        const float least = low != low ? -__builtin_inff() : low;
        auto push = [&](float v, int64_t i) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kList) sh.list[at] = argmax_key(v, (int32_t)i);
        };
#pragma unroll
        for (int t = 0; t < kTiles; t++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int64_t i = first + t * (kThreads * 8) + j;
                if (__builtin_amdgcn_ballot_w64(x[t][j] >= least) != 0 && x[t][j] >= least && i >= 0 && i < a.vocab) push(x[t][j], i);
            }
        __syncthreads();
        int n = sh.count;
        if (n > kList) {
            // too many (equal or nearly equal logits): the exact top-th largest order
            // bits, bit by bit over all logits, then the greater ones and of the equal
            // ones as many as are missing, lowest index first
            unsigned nth = 0;
            for (int b = 31; b >= 0; b--) {
                const unsigned tr = nth | (1u << b);
                int k = 0;
#pragma unroll
                for (int t = 0; t < kTiles; t++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int64_t i = first + t * (kThreads * 8) + j;
                        k += x[t][j] == x[t][j] && i >= 0 && i < a.vocab && order_bits(x[t][j]) >= tr;
                    }
                k = wave_sum_i32(k);
                __syncthreads();
                if (lane == 0) sh.wave_count[wave] = k;
                __syncthreads();
                if (sh.wave_count[0] + sh.wave_count[1] + sh.wave_count[2] + sh.wave_count[3] >= a.top) nth = tr;
            }
            __syncthreads();
            if (tid == 0) sh.count = 0;
            __syncthreads();
#pragma unroll
            for (int t = 0; t < kTiles; t++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int64_t i = first + t * (kThreads * 8) + j;
                    if (x[t][j] == x[t][j] && i >= 0 && i < a.vocab && order_bits(x[t][j]) > nth) push(x[t][j], i);
                }
            __syncthreads();
            int have = sh.count;   // below top
#pragma unroll
            for (int t = 0; t < kTiles; t++) {
                int k = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int64_t i = first + t * (kThreads * 8) + j;
                    k += x[t][j] == x[t][j] && i >= 0 && i < a.vocab && order_bits(x[t][j]) == nth;
                }
                // equal logits in front of this thread's, in the tile
                int before = k;
                for (int o = 1; o < 64; o <<= 1) {
                    const int up = __shfl_up(before, o);
                    if (lane >= o) before += up;
                }
                __syncthreads();
                if (lane == 63) sh.wave_count[wave] = before;
                __syncthreads();
                before -= k;
                int all = 0;
                for (int w = 0; w < 4; w++) {
                    if (w < wave) before += sh.wave_count[w];
                    all += sh.wave_count[w];
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int64_t i = first + t * (kThreads * 8) + j;
                    if (x[t][j] == x[t][j] && i >= 0 && i < a.vocab && order_bits(x[t][j]) == nth) {
                        if (have + before < a.top) sh.list[have + before] = argmax_key(x[t][j], (int32_t)i);
                        before++;
                    }
                }
                have += all;
            }
            __syncthreads();
            n = min(have, a.top);
        }
        rank_list(sh, n, a.top);
    } else {
        __syncthreads();
    }

    Part p;
    p.m = m;
    p.s = (sh.red[0] + sh.red[1]) + (sh.red[2] + sh.red[3]);
    p.t = (sh.red[4] + sh.red[5]) + (sh.red[6] + sh.red[7]);
    p.pad = 0.0f;
    if (parts == 1) {
        finish_row(a, row, p, sh.best);
        return;
    }
    Part* ps = (Part*)a.scratch;
    unsigned long long* ks = (unsigned long long*)(ps + (int64_t)a.rows * parts);
    if (tid == 0) ps[row * parts + part] = p;
    for (int i = tid; i < a.top; i += kThreads) ks[(row * parts + part) * a.top + i] = sh.best[i];
}

__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogprobsArgs a, int parts) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.x;
    const Part* ps = (const Part*)a.scratch + row * parts;
    const unsigned long long* ks = (const unsigned long long*)((const Part*)a.scratch + (int64_t)a.rows * parts) + row * parts * a.top;
    const int lane = lane_id();
    // every wavefront for itself
    float m = -__builtin_inff();
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, ps[i].m);
    m = wave_max_f32(m);
    float s = 0.0f, t = 0.0f;
    for (int i = lane; i < parts; i += 64) {
        const Part p = ps[i];
        if (p.m == -__builtin_inff() && p.s == 0.0f) continue;   // nothing but minus infinity
        const float y = (p.m - m) * kLog2e, e = __builtin_amdgcn_exp2f(y);
        s += e * p.s;
        t += e * __builtin_fmaf(fmaxf(y, -1e30f), p.s, p.t);
    }
    Part p;
    p.m = m;
    p.s = wave_butterfly_sum(s);
    p.t = wave_butterfly_sum(t);
    p.pad = 0.0f;
    // the parts' keys, in rounds of what the list holds behind the best so far
    const int64_t all = (int64_t)parts * a.top;
    int kept = 0;
    for (int64_t at = 0; at < all;) {
        const int take = (int)min((int64_t)(kList - kept), all - at);
        if ((int)threadIdx.x < kept) sh.list[threadIdx.x] = sh.best[threadIdx.x];
        for (int i = threadIdx.x; i < take; i += kThreads) sh.list[kept + i] = ks[at + i];
        __syncthreads();
        rank_list(sh, kept + take, a.top);
        at += take;
        kept = a.top;
    }
    finish_row(a, row, p, sh.best);
}

}  // namespace

size_t logprobs_scratch(int32_t rows, int32_t vocab, int32_t top) {
    const int64_t parts = parts_of(vocab);
    return parts <= 1 ? 0 : (size_t)rows * parts * (sizeof(Part) + (size_t)top * 8);
}

hipError_t launch_token_logprobs(hipStream_t s, const LogprobsArgs& a) {
    if (a.rows <= 0) return hipSuccess;
    const int parts = (int)parts_of(a.vocab);
    const dim3 grid(a.rows, parts), block(kThreads);
    if (a.dtype == DT_F32) TL_KLAUNCH((logprobs_kernel<DT_F32>), grid, block, 0, s, a, parts);
    else if (a.dtype == DT_BF16) TL_KLAUNCH((logprobs_kernel<DT_BF16>), grid, block, 0, s, a, parts);
    else TL_KLAUNCH((logprobs_kernel<DT_F16>), grid, block, 0, s, a, parts);
    if (parts > 1) TL_KLAUNCH(logprobs_join_kernel, dim3(a.rows), block, 0, s, a, parts);
    return hipGetLastError();
}

}  // namespace tl
