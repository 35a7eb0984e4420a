// tl_score.hip -- log probability of a given token, entropy and the most probable
// alternatives of each row of logits, in one pass over the logits.
//
// With m = max x, S = sum e^(x - m), T = sum (x - m) e^(x - m):
//   log p_i = x_i - m - ln S,   H = ln S - T / S.
// A workgroup takes a part of a row into registers (32 logits per thread, 8 where
// there are few rows), leaves its m, S, T (base 2) and at least its largest `top`
// logits; the workgroup of a row that is done last joins the parts, or a second
// kernel.  A row of one part is finished by its own workgroup.
//
// Alternatives are ordered by logit, equal ones by index: 64-bit keys (the
// order-preserving bits of the logit above, the index's complement below), so
// the order is total.  A workgroup does not sort: the top-th largest of the
// maxima of its 64 sets of logits is a lower bound of the top-th largest logit,
// and the few logits above it are ranked against each other.
//
// What bounds it: 500 rows of 100003 bfloat16 logits with 20 alternatives take 33.8
// us (3.0 TB/s), 29 of them in the first kernel, whose vector instructions (some 450
// a wavefront, 32 of them exponentials at a quarter of the rate) fill most of its
// time: reading alone would take 14.5.  Without alternatives it is 21.9 us.  So the
// registers are held to 72, for 7 wavefronts on a SIMD (6: 35.3 us; 8 spill: 47),
// all loads of a wavefront are issued at once, a part's candidates are not ranked but
// handed to the join (2.4 us less), and logits are compared with the bound only where
// the largest of four reaches it.  One row of 32000: 7.2 us.
//
// Exponentials and logarithms are the hardware's, base 2: log probabilities are off by
// 6e-8 to 1e-7 of themselves (norms over the rows, against 64 bits), where float32
// functions leave 5e-8.
#include <algorithm>

#include "tl_rows.h"

namespace tl {
namespace {

constexpr int kThreads = 256;
constexpr int kRun = kThreads * 8;                 // 8 adjacent logits per thread and tile
constexpr int kMostTiles = 4;
constexpr int kList = 1024;                        // candidates ranked at once
// Rows in parts of up to 8192 logits if that makes 256 workgroups, else of 2048: 32
// rows of 32000 (bf16 and float32 alike) 8.4 us against 9.2, 64 rows 11.2 against
// 10.3.  Parts are joined in place, by the last workgroup of a row, in launches of up to
// 512: its store, wait and count cost each workgroup time, hidden where all run at once
// (one row of 32000: 7.2 us in one kernel, one launch less); 500 rows of 100003 take
// 49.7 us so and 37.9 with a kernel for the join.
constexpr int64_t kEnough = 256, kJoinInPlace = 512;
constexpr float kLn2 = 0.693147180559945309417f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;        // the least finite float

typedef unsigned long long u64;
typedef u64 v2u64 __attribute__((ext_vector_type(2)));

TL_DEV unsigned order_bits(float v) {              // greater logits, greater bits; never 0
    if (v == 0.0f) v = 0.0f;                       // -0 and +0 are equal
    const unsigned u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// s, t relative to m, in base 2: s = sum 2^y, t = sum y 2^y, y = (x - m) log2 e
struct Part {
    float m, s, t;
};

struct Shared {
    unsigned set_max[64];
    float red[8];
    int count, last;
    int wave_count[4];
    alignas(16) u64 list[kList + 8];
    u64 best[kMaxTop];
};

// A part in scratch is 2 + kept_of(top) words: m and s, t, its keys in any order (0:
// none).  Other workgroups read them, so they go past the caches: loads and stores of
// agent scope.  With room for some more than `top` keys the candidates of most parts
// go there as they are, to be ranked once by the join; more than that are ranked first.
TL_HD inline int kept_of(int top) { return top > 0 ? top + 12 : 0; }
TL_DEV void part_store(u64* p, u64 v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
TL_DEV u64 part_load(const u64* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
TL_DEV u64 two(float lo, float hi) { return (u64)__float_as_uint(hi) << 32 | __float_as_uint(lo); }

// The greatest number with 16 leading bits that at least `top` of the 64 lanes reach:
// no greater than the top-th largest of any keys of which the lanes hold some.
TL_DEV unsigned bound_of(unsigned key, int top) {
    unsigned bound = 0;
#pragma unroll
    for (int b = 31; b >= 16; b--) {
        const unsigned c = bound | (1u << b);
        if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= c)) >= top) bound = c;
    }
    return bound;
}

// list[0 .. n) (distinct keys, 0: none) ranked; the largest `top` to best[] in order
TL_DEV void rank_list(Shared& sh, int n, int top) {
    const int tid = threadIdx.x;
    if (tid < 8) sh.list[n + tid] = 0ull;
    if (tid < top) sh.best[tid] = 0ull;
    if (n > 64) __syncthreads();      // (fewer are one wavefront's work)
    for (int i = tid; i < n; i += kThreads) {
        const u64 k = sh.list[i];
        int r = 0;
        for (int j = 0; j < n; j += 8) {
            v2u64 q[4];
#pragma unroll
            for (int c = 0; c < 4; c++) q[c] = *(const v2u64*)&sh.list[j + 2 * c];
#pragma unroll
            for (int c = 0; c < 4; c++) r += (int)(q[c][0] > k) + (int)(q[c][1] > k);
        }
        if (k != 0ull && r < top) sh.best[r] = k;
    }
    __syncthreads();
}

// Of list[0 .. n), n <= kList, those that may be among the largest `top`, in any order.
// The whole workgroup takes part; every wavefront's keys are in the list.
TL_DEV int thin_list(Shared& sh, int n, int top) {
    const int tid = threadIdx.x;
    u64 k[kList / kThreads];
    u64 most = 0;
#pragma unroll
    for (int j = 0; j < kList / kThreads; j++) {
        k[j] = tid + j * kThreads < n ? sh.list[tid + j * kThreads] : 0ull;
        most = max(most, k[j]);
    }
    unsigned m = (unsigned)(most >> 32);
    m = max(m, (unsigned)dpp<kDppXor1>((int)m));
    m = max(m, (unsigned)dpp<kDppXor2>((int)m));
    if ((tid & 3) == 0) sh.set_max[tid >> 2] = m;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const unsigned bound = max(1u, bound_of(sh.set_max[lane_id()], top));
#pragma unroll
    for (int j = 0; j < kList / kThreads; j++)
        if ((unsigned)(k[j] >> 32) >= bound) sh.list[atomicAdd(&sh.count, 1)] = k[j];
    __syncthreads();
    return sh.count;
}

// what a row gives, from its m, S, T and its best keys; target: targets[row], xt: its logit
TL_DEV void finish_row(const LogprobsArgs& a, int64_t row, const Part& p, const u64* best, int target, float xt) {
    const float ls = __log2f(p.s);
    if (threadIdx.x == 0) {
        float lp = 0.0f;
        if (target >= a.vocab) {
            lp = __builtin_nanf("");
            if (a.fault) *a.fault = 1;
        } else if (target >= 0) {
            lp = (xt - p.m) - ls * kLn2;
        }
        a.logprob[row] = lp;
        if (a.entropy) a.entropy[row] = (ls - p.t / p.s) * kLn2;
    }
    if ((int)threadIdx.x < a.top) {
        const u64 k = best[threadIdx.x];
        const int64_t at = row * a.top + threadIdx.x;
        a.top_ids[at] = k ? key_index(k) : -1;
        a.top_logprobs[at] = k ? (key_logit(k) - p.m) - ls * kLn2 : __builtin_nanf("");
    }
}

TL_DEV float target_logit(const LogprobsArgs& a, int64_t row, int target) {
    return target >= 0 && target < a.vocab ? load1(a.logits, row * a.stride + target, a.dtype) : 0.0f;
}

// the parts of a row joined by one workgroup
TL_DEV void join_row(const LogprobsArgs& a, int64_t row, int parts, int target, Shared& sh) {
    const int each = kept_of(a.top), words = 2 + each, tid = threadIdx.x, lane = lane_id();
    const u64* from = (const u64*)a.scratch + row * parts * words;
    const float xt = target_logit(a, row, target);
    // the parts' keys, in rounds of what the list holds behind the best so far
    const int64_t all = (int64_t)parts * each;
    int kept = 0;
    for (int64_t at = 0; at < all;) {
        const int take = (int)min((int64_t)(kList - kept), all - at);
        u64 k[kList / kThreads];
#pragma unroll
        for (int j = 0; j < kList / kThreads; j++) {
            const unsigned i = (unsigned)(at + min(tid + j * kThreads, take - 1));
            const unsigned part = i / (unsigned)each;
            k[j] = part_load(from + (int64_t)part * words + 2 + (i - part * each));
        }
        if (tid < kept) sh.list[tid] = sh.best[tid];
#pragma unroll
        for (int j = 0; j < kList / kThreads; j++)
            if (tid + j * kThreads < take) sh.list[kept + tid + j * kThreads] = k[j];
        __syncthreads();
        const int n = thin_list(sh, kept + take, a.top);
        rank_list(sh, n, a.top);
        at += take;
        kept = a.top;
    }
    // every wavefront for itself
    float m = -__builtin_inff();
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, __uint_as_float((unsigned)part_load(from + (int64_t)i * words)));
    m = wave_max_f32(m);
    float s = 0.0f, t = 0.0f;
    for (int i = lane; i < parts; i += 64) {
        const u64 ms = part_load(from + (int64_t)i * words);
        const float pm = __uint_as_float((unsigned)ms), ps = __uint_as_float((unsigned)(ms >> 32));
        const float pt = __uint_as_float((unsigned)part_load(from + (int64_t)i * words + 1));
        if (pm == -__builtin_inff() && ps == 0.0f) continue;   // nothing but minus infinity
        const float y = (pm - m) * kLog2e, e = __builtin_amdgcn_exp2f(y);
        s += e * ps;
        t += e * __builtin_fmaf(fmaxf(y, -1e30f), ps, pt);
    }
    Part p;
    p.m = m;
    p.s = wave_butterfly_sum(s);
    p.t = wave_butterfly_sum(t);
    finish_row(a, row, p, sh.best, target, xt);
}

template <int DT, int TILES>
__global__ __launch_bounds__(kThreads, TILES == 1 ? 4 : 7) void logprobs_kernel(LogprobsArgs a, int parts, int tiles) {
    __shared__ Shared sh;
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    const int64_t row = blockIdx.x / (unsigned)parts;
    const int part = (int)(blockIdx.x - (unsigned)row * parts);
    const char* base = (const char*)a.logits + row * a.stride * ES;
    // units of 8 start at multiples of 16 bytes: the row's first logit is at place
    // `skew` of unit 0
    const int skew = (int)((uintptr_t)base / ES & (16 / ES - 1));
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
    int first = part * (kRun * tiles) + tid * 8 - skew;   // this thread's first index
    const int live = min(tiles, (a.vocab + skew - part * (kRun * tiles) + kRun - 1) / kRun);
    const int target = a.targets[row];
    if (tid == 0) sh.count = 0;

    // whole units first, all on their way at once; then the row's ends, one by one
    v4i raw[TILES][ES / 2];
    constexpr int kNone = DT == DT_F32 ? (int)0xFF800000 : DT == DT_BF16 ? (int)0xFF80FF80 : (int)0xFC00FC00;   // minus infinities
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        const int i = first + t * kRun;
#pragma unroll
        for (int h = 0; h < ES / 2; h++) raw[t][h] = v4i{kNone, kNone, kNone, kNone};
        if (t < live && i >= 0 && i + 8 <= a.vocab)
#pragma unroll
            for (int h = 0; h < ES / 2; h++) raw[t][h] = __builtin_nontemporal_load((const v4i*)(base + (int64_t)i * ES) + h);
    }
    float x[TILES][8];
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v4f q;
            if constexpr (DT == DT_F32) q = __builtin_bit_cast(v4f, raw[t][h]);
            else q = unpack4(v2i{raw[t][0][2 * h], raw[t][0][2 * h + 1]}, DT);
#pragma unroll
            for (int j = 0; j < 4; j++) x[t][4 * h + j] = q[j];
        }
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        const int i = first + t * kRun;
        if (t >= live) break;
        if ((i < 0 && i + 8 > 0) || (i < a.vocab && i + 8 > a.vocab)) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j >= 0 && i + j < a.vocab) x[t][j] = load1(base, i + j, DT);
        }
    }

    // nothing computed from the logits is kept in registers past this
    auto fresh = [&] {
#pragma unroll
        for (int t = 0; t < TILES; t++)
#pragma unroll
            for (int j = 0; j < 8; j++) asm volatile("" : "+v"(x[t][j]));
        asm volatile("" : "+v"(first));
    };

    // maximum of the workgroup, and of each set of 4 threads
    float own = -__builtin_inff(), most[TILES][2];   // (NaN are not maxima)
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            most[t][h] = fmaxf(fmaxf(x[t][4 * h], x[t][4 * h + 1]), fmaxf(x[t][4 * h + 2], x[t][4 * h + 3]));
            own = fmaxf(own, most[t][h]);
        }
    float mx = fmaxf(own, lane_xor<1>(own));
    mx = fmaxf(mx, lane_xor<2>(mx));
    if ((lane & 3) == 0) sh.set_max[wave * 16 + (lane >> 2)] = __float_as_uint(mx);
    __syncthreads();
    const float set = __uint_as_float(sh.set_max[lane]);
    const float m = wave_max_f32(set);

    u64 key = 0ull;   // of this thread, for the part's words
    if (a.top > 0) {
        // the bound as a logit, finite: bound's lower bits are zero, for a negative one the
        // lowest of its class
        const unsigned bound = bound_of(order_bits(set), a.top);
        const float low = __uint_as_float(bound & 0x80000000u ? bound & 0x7FFFFFFFu : ~bound);
        const float least = low >= kLowest ? low : kLowest;
        if (__builtin_amdgcn_ballot_w64(own >= least) != 0) {
#pragma unroll
            for (int t = 0; t < TILES; t++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (t >= live || __builtin_amdgcn_ballot_w64(most[t][h] >= least) == 0) continue;
#pragma unroll
                    for (int j = 4 * h; j < 4 * h + 4; j++)
                        if (__builtin_amdgcn_ballot_w64(x[t][j] >= least) != 0 && x[t][j] >= least) {
                            const int at = atomicAdd(&sh.count, 1);
                            if (at < kList) sh.list[at] = argmax_key(x[t][j], first + t * kRun + j);
                        }
                }
        }
        __syncthreads();
        int n = sh.count;
        if (n > kList || n < a.top) {
            // Too many (equal or nearly equal logits): the exact top-th largest order bits, bit
            // by bit over all logits, and the greater ones.  Too few (the others are minus
            // infinity): all of them.  Then of the equal ones, or of minus infinity, as many
            // as are missing, lowest index first.
            unsigned nth = order_bits(-__builtin_inff());
            auto bits = [&](int t, int j) {   // 0: no logit (a tile behind the part's last has the next part's indices)
                const int i = first + t * kRun + j;
                return t < live && x[t][j] == x[t][j] && (unsigned)i < (unsigned)a.vocab ? order_bits(x[t][j]) : 0u;
            };
            if (n > kList) {
                nth = 0;
                for (int b = 31; b >= 0; b--) {
                    const unsigned tr = nth | (1u << b);
                    int k = 0;
                    fresh();
#pragma unroll
                    for (int t = 0; t < TILES; t++)
#pragma unroll
                        for (int j = 0; j < 8; j++) k += bits(t, j) >= tr;
                    k = wave_sum_i32(k);
                    __syncthreads();
                    if (lane == 0) sh.wave_count[wave] = k;
                    __syncthreads();
                    if (sh.wave_count[0] + sh.wave_count[1] + sh.wave_count[2] + sh.wave_count[3] >= a.top) nth = tr;
                }
                __syncthreads();
                if (tid == 0) sh.count = 0;
                __syncthreads();
                fresh();
#pragma unroll
                for (int t = 0; t < TILES; t++)
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (bits(t, j) > nth) sh.list[atomicAdd(&sh.count, 1)] = argmax_key(x[t][j], first + t * kRun + j);
                __syncthreads();
            }
            int have = sh.count;   // below top
            fresh();
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                int k = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) k += bits(t, j) == nth;
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
                for (int j = 0; j < 8; j++)
                    if (bits(t, j) == nth) {
                        if (have + before < a.top) sh.list[have + before] = argmax_key(x[t][j], first + t * kRun + j);
                        before++;
                    }
                have += all;
            }
            __syncthreads();
            n = min(have, a.top);
        }
        if (parts > 1 && n <= kept_of(a.top)) {
            if (tid >= 2 && tid - 2 < n) key = sh.list[tid - 2];
        } else {
            rank_list(sh, n, a.top);
            if (tid >= 2 && tid - 2 < a.top) key = sh.best[tid - 2];
        }
    }

    // Sums relative to the workgroup's maximum, y = x log2 e - m2 in one rounding; m2 is
    // m log2 e but for `rest`.  Where that is not small (|m| > 4096) x - m comes first.  A
    // logit of minus infinity adds nothing.
    const bool far = !(fabsf(m) <= 4096.0f);
    if (far) {
        const float off = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int t = 0; t < TILES; t++)
#pragma unroll
            for (int j = 0; j < 8; j++) x[t][j] -= off;
    }
    const float m2 = far ? 0.0f : m * kLog2e;
    const float rest = far ? 0.0f : __builtin_fmaf(m, kLog2e, -m2);
    float s = 0.0f, tt = 0.0f;
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        if (t >= live) break;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float y = __builtin_fmaf(x[t][j], kLog2e, -m2);
            const float e = __builtin_amdgcn_exp2f(y);
            s += e;
            tt = __builtin_fmaf(fmaxf(y, -1e30f), e, tt);
        }
    }
    s = wave_butterfly_sum(s);
    tt = wave_butterfly_sum(tt);
    if (lane == 0) {
        sh.red[wave] = s;
        sh.red[4 + wave] = tt;
    }
    __syncthreads();
    Part p;
    const float scale = __builtin_amdgcn_exp2f(-rest);
    p.m = m;
    p.s = ((sh.red[0] + sh.red[1]) + (sh.red[2] + sh.red[3])) * scale;
    p.t = ((sh.red[4] + sh.red[5]) + (sh.red[6] + sh.red[7])) * scale - rest * p.s;
    if (parts == 1) {
        finish_row(a, row, p, sh.best, target, target_logit(a, row, target));
        return;
    }
    const int words = 2 + kept_of(a.top);
    u64* to = (u64*)a.scratch + (row * parts + part) * words;
    if (tid < words) part_store(to + tid, tid == 0 ? two(p.m, p.s) : tid == 1 ? two(p.t, 0.0f) : key);
    if (!a.counters) return;
    // the stores have arrived before the part is counted
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const int got = __hip_atomic_fetch_add(a.counters + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.last = got == parts - 1;
        if (sh.last) __hip_atomic_store(a.counters + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (sh.last) join_row(a, row, parts, target, sh);
}

__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogprobsArgs a, int parts) {
    __shared__ Shared sh;
    join_row(a, blockIdx.x, parts, a.targets[blockIdx.x], sh);
}

// How a row is cut: parts of up to kMostTiles tiles, as even as they come.  Where
// those are few for the card, one tile each if one round of the join takes them.
struct Cut {
    int tiles, parts;
};
Cut cut_of(int32_t rows, int32_t vocab, int32_t top) {
    const int all = (int)(((int64_t)vocab + 7 + kRun - 1) / kRun);   // (a row may start up to 7 places into its first unit)
    const int parts = (all + kMostTiles - 1) / kMostTiles;
    if ((int64_t)rows * parts < kEnough && all * kept_of(top) <= kList) return {1, all};
    const int tiles = (all + parts - 1) / parts;
    return {tiles, (all + tiles - 1) / tiles};
}

}  // namespace

int64_t logprobs_workgroups(int32_t rows, int32_t vocab, int32_t top) { return (int64_t)rows * cut_of(rows, vocab, top).parts; }

size_t logprobs_scratch(int32_t rows, int32_t vocab, int32_t top) {
    const Cut c = cut_of(rows, vocab, top);
    return c.parts <= 1 ? 0 : (size_t)rows * c.parts * (2 + kept_of(top)) * 8;
}

hipError_t launch_token_logprobs(hipStream_t s, const LogprobsArgs& in) {
    if (in.rows <= 0) return hipSuccess;
    LogprobsArgs a = in;
    const Cut c = cut_of(a.rows, a.vocab, a.top);
    if (a.rows > kOpCounters || (int64_t)a.rows * c.parts > kJoinInPlace) a.counters = nullptr;
    const dim3 grid((unsigned)(a.rows * c.parts)), block(kThreads);
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (c.tiles == 1) TL_KLAUNCH((logprobs_kernel<DT, 1>), grid, block, 0, s, a, c.parts, c.tiles);
        else TL_KLAUNCH((logprobs_kernel<DT, kMostTiles>), grid, block, 0, s, a, c.parts, c.tiles);
    };
    using std::integral_constant;
    if (a.dtype == DT_F32) go(integral_constant<int, DT_F32>{});
    else if (a.dtype == DT_BF16) go(integral_constant<int, DT_BF16>{});
    else go(integral_constant<int, DT_F16>{});
    if (c.parts > 1 && !a.counters) TL_KLAUNCH(logprobs_join_kernel, dim3(a.rows), block, 0, s, a, c.parts);
    return hipGetLastError();
}

}  // namespace tl
