// One token per logits row from given uniform numbers (sm_100a): temperature,
// top-k, min-p and top-p on the integer weights of the library's sampling rule
// (fl_sample.cuh), so every sum is exact and the draw does not depend on the
// order of any reduction. The rule is stated at fl_cuda_sample in
// include/fl_cuda.h.
//
// A row is held by one CTA, or by a cluster of up to eight: every thread reads
// 64 tokens at most, once, turns them into weights and keeps those in
// registers. A threshold (of top-k by count, of top-p by mass) is found by
// bisection between weights lo and hi, near their geometric mean: passes over
// the registers until 128 weights are undecided, and those are compared all
// with all at once. Counts and masses share one 64-bit word (44 bits of mass).
// The draw is a prefix sum in token order: over the warps, each of which holds
// a contiguous piece of the row, then within the one the target falls into.
// 448 rows of 32064 with mixed rules take 73 us, of which instructions are about 31
// (25 a token for its weight, 3 for each of about 18 passes): one CTA fills an SM's
// registers, so that nothing runs while its warps reduce and meet, and 448 rows are 3.03
// waves. Few warps with much work each, because a pass costs apart from that
// the warps' reductions (32 tokens a thread of 1024 took 85 us). One row takes 18 us
// and 61 rows of 128011 in 16 bits 104, most of it cluster barriers.
#include <float.h>
#include <limits.h>

#include <algorithm>

#include "fl_common.cuh"
#include "fl_kernels.h"
#include "fl_kv8_types.cuh"
#include "fl_runtime.h"
#include "fl_sample.cuh"

namespace fl {

namespace {

typedef unsigned __int128 u128;
typedef unsigned long long u64;
constexpr int kTok = 64;          // tokens per thread
constexpr int kPairs = 128;       // undecided weights compared all with all
// In a register a weight carries a count of one above its 24 bits (and the
// value 2^24): eight of them add up in one word, count and mass at once.
constexpr uint32_t kTag = 1u << 28;
constexpr int kMassBits = 44;
constexpr u64 kMass = (1ull << kMassBits) - 1;
// The weight of a larger logit is smaller, by one, for 2878 of all floats below 0
// (each against the float before it), with weights from kUnorderedMin to kUnorderedMax:
// the polynomial's last roundings. tests/sample_weight_check.c goes through all floats.
constexpr uint32_t kUnorderedMin = 13066122u, kUnorderedMax = 16518617u;

struct SampleArgs {
    const void* logits;
    size_t ld;
    int V, seg;                   // tokens of a CTA of the row's cluster
    int rows, ahead;              // rows; how many later the row that an SM takes next
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* tokens;
};

// A logit as the rule reads it: NaN counts as -inf, +inf as the largest float.
__device__ __forceinline__ float canon(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }
template <int DT>
__device__ __forceinline__ float logit(const void* l, int i) {
    if constexpr (DT == FL_F32) return canon(static_cast<const float*>(l)[i]);
    else if constexpr (DT == FL_F16) return canon(__half2float(static_cast<const __half*>(l)[i]));
    else return canon(__bfloat162float(static_cast<const __nv_bfloat16*>(l)[i]));
}
// Orders floats as unsigned integers, -0 as 0.
__device__ __forceinline__ uint32_t sortable(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unsortable(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
// trunc(p 2^24) within [0, 2^24]; 0 for NaN.
__device__ __forceinline__ uint32_t fixed24(float p) {
    return __float2uint_rz(__fmul_rn(fminf(fmaxf(p, 0.0f), 1.0f), 16777216.0f));
}

// Hides that x is what it was, so that a loop over the registers that uses it
// is computed again where it stands: kept for later, its 64 results would
// push the weights out of the registers.
__device__ __forceinline__ void again(uint32_t& x) { asm volatile("" : "+r"(x)); }

// sum += w where w >= t. The add is a multiply-add by a one that the compiler
// does not see: it runs beside the comparison in the other pipe, which an add
// would share (a pass over the registers took 40 % less).
__device__ __forceinline__ void add_if_ge(uint32_t& sum, uint32_t w, uint32_t t, uint32_t one) {
    asm("{\n\t.reg .pred p;\n\tsetp.ge.u32 p, %1, %2;\n\t@p mad.lo.u32 %0, %1, %3, %0;\n\t}"
        : "+r"(sum)
        : "r"(w), "r"(t), "r"(one));
}

// A count in the upper 20 bits and a mass in the lower 44 of a word.
__device__ __forceinline__ u64 pack(u64 count, u64 mass) { return (count << kMassBits) + mass; }

// Sum over the warp of at most 64 weights a lane (c of them, together m < 2^31), packed.
__device__ __forceinline__ u64 warp_pack(uint32_t c, uint32_t m) {
    const uint32_t a = __reduce_add_sync(0xffffffffu, m & 0xfffffu);
    const uint32_t b = __reduce_add_sync(0xffffffffu, (m >> 20) | c << 16);
    return pack(b >> 16, ((u64)(b & 0xffffu) << 20) + a);
}

// Reductions and prefix sums over the threads of a row's CTA or cluster.
template <int NT, int CL>
struct Row {
    static constexpr int NW = NT / 32, NS = CL * NW, cl = CL;
    struct Shared {
        u64 slot[2][NS];
        uint32_t pairs[kPairs];
        uint32_t own[CL > 1 ? kPairs : 1];   // this CTA's part of them
        int n;
    };
    Shared& sm;
    int lane, warp, rank, me;   // me: this warp among all of the row
    int phase = 0;
    uint32_t one = 1u;

    __device__ Row(Shared& s) : sm(s), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), rank(0) {
        if (CL > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        me = rank * NW + warp;
        asm volatile("" : "+r"(one));
        if (CL > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA has started
    }
    // Before the first access to another CTA's shared memory: every CTA of the
    // cluster has to have started.
    __device__ __forceinline__ void started() {
        if constexpr (CL > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    }
    __device__ __forceinline__ void sync() {
        if constexpr (CL > 1)
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else
            __syncthreads();
    }
    // Every warp's v (the same in its lanes) to all threads: read slots() after
    // it. Two sets of slots in turn: a warp that is a pass ahead writes the other.
    __device__ __forceinline__ const u64* share(u64 v) {
        u64* p = &sm.slot[phase][me];
        if constexpr (CL > 1) {
            if (lane < CL) {
                uint32_t ra;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                             : "=r"(ra)
                             : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(lane));
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(ra), "l"(v) : "memory");
            }
        } else if (lane == 0) {
            *p = v;
        }
        sync();
        const u64* s = sm.slot[phase];
        phase ^= 1;
        return s;
    }
    __device__ __forceinline__ u64 sum(uint32_t c, uint32_t m) {
        const u64* s = share(warp_pack(c, m));
        u64 t = 0;
#pragma unroll
        for (int i = 0; i < NS; i++) t += s[i];
        return t;
    }
    __device__ __forceinline__ uint32_t max32(uint32_t v) {
        const u64* s = share(__reduce_max_sync(0xffffffffu, v));
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < NS; i++) t = max(t, (uint32_t)s[i]);
        return t;
    }
    // v to the same place in every CTA of the cluster
    __device__ __forceinline__ void store_all(uint32_t* p, uint32_t v) {
        if constexpr (CL > 1) {
            const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
#pragma unroll
            for (int i = 0; i < CL; i++) {
                uint32_t ra;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(a), "r"(i));
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ra), "r"(v) : "memory");
            }
        } else {
            *p = v;
        }
    }
};

// Sum of the row's weights at or above t.
template <class R>
__device__ __forceinline__ u64 at_least(R& row, const uint32_t (&w)[kTok], uint32_t t) {
    const uint32_t tt = t + kTag;
    uint32_t m = 0, c = 0;   // 64 weights of at most 2^24 sum to 2^30 at most
#pragma unroll
    for (int i = 0; i < kTok; i += 8) {
        uint32_t g = 0;
#pragma unroll
        for (int j = i; j < i + 8; j++) add_if_ge(g, w[j], tt, row.one);
        c += g >> 28;
        m += g & (kTag - 1u);
    }
    return row.sum(c, m);
}

// The largest t in [lo, hi) with ok(sum of the weights >= t), given that
// ok holds at lo and not at hi; slo and shi are those sums, and on return the
// ones at t and t + 1.
template <class R, class Ok>
__device__ __forceinline__ uint32_t bisect(R& row, const uint32_t (&w)[kTok], uint32_t lo, uint32_t hi, u64& slo,
                                           u64& shi, Ok ok) {
    while (hi - lo > 1u && (slo - shi) >> kMassBits > kPairs) {
        // the mean of their logarithms, roughly (of their float patterns)
        const uint32_t b = (__float_as_uint(__uint2float_rz(lo)) + __float_as_uint(__uint2float_rz(hi))) / 2u;
        const uint32_t mid = min(max(__float2uint_rz(__uint_as_float(b)), lo + 1u), hi - 1u);
        const u64 s = at_least(row, w, mid);
        if (ok(s)) { lo = mid; slo = s; } else { hi = mid; shi = s; }
    }
    if (hi - lo <= 1u) return lo;
    // the undecided weights of the whole row in every CTA, each against all of
    // them: the threshold is the largest at which ok holds. A call may come here
    // without a pass, while other warps still sum the pairs of the call before.
    __syncthreads();
    for (int i = threadIdx.x; i < kPairs; i += R::NW * 32) row.sm.pairs[i] = 0u;
    if (threadIdx.x == 0) row.sm.n = 0;
    __syncthreads();
    uint32_t* list = row.cl > 1 ? row.sm.own : row.sm.pairs;
    const uint32_t from = lo + kTag, span = hi - lo;
#pragma unroll
    for (int i = 0; i < kTok; i++)   // in any order: their sums are exact
        if (w[i] - from < span) list[atomicAdd(&row.sm.n, 1)] = w[i] - kTag;
    __syncthreads();
    if constexpr (R::cl > 1) {
        const int n = row.sm.n;
        const u64* s = row.share(row.warp == 0 ? n : 0);
        int at = 0;
#pragma unroll
        for (int i = 0; i < R::NS; i++) at += i < row.me - row.warp ? (int)s[i] : 0;
        if (threadIdx.x < n) row.store_all(&row.sm.pairs[at + threadIdx.x], row.sm.own[threadIdx.x]);
        row.sync();
    }
    constexpr int TP = R::NW * 32 / kPairs;   // threads per weight
    const uint32_t mine = row.sm.pairs[threadIdx.x / TP];
    auto sums = [&](uint32_t t, bool strictly) -> u64 {   // of the pairs, by the TP threads of a weight
        uint32_t c = 0, m = 0;   // 128 weights below 2^24, or equal to it: 2^31 at most
#pragma unroll 8
        for (int i = threadIdx.x % TP; i < kPairs; i += TP) {
            const uint32_t f = row.sm.pairs[i];
            const bool in = strictly ? f > t : f >= t;
            m += in ? f : 0u;
            c += in;
        }
#pragma unroll
        for (int o = 1; o < TP; o <<= 1) {
            c += __shfl_xor_sync(0xffffffffu, c, o);
            m += __shfl_xor_sync(0xffffffffu, m, o);
        }
        return pack(c, m);
    };
    const u64 base = shi;
    const u64 at_mine = base + sums(mine, false);   // by every thread: its shuffles need whole warps
    const uint32_t t = max(lo, row.max32(mine >= lo && ok(at_mine) ? mine : 0u));
    slo = base + sums(t, false);
    shi = base + sums(t, true);
    return t;
}

template <int DT, int NT, int CL>
__global__ void __launch_bounds__(NT, NT >= 512 ? 1 : 512 / NT) sample_rows_kernel(const SampleArgs a) {
    typedef Row<NT, CL> R;
    constexpr int ES = DT == FL_F32 ? 4 : 2, VEC = 16 / ES, J = kTok / VEC;
    __shared__ typename R::Shared shared;
    R row(shared);
    const int r = blockIdx.x / CL;
    const char* l = static_cast<const char*>(a.logits) + (size_t)r * a.ld * ES;
    const int V = a.V;
    const int i0 = row.rank * a.seg, i1 = min(V, i0 + a.seg);   // this CTA's tokens
    // token of (group j, element e) of this thread: a warp's tokens are a
    // contiguous piece, groups of VEC begin on 16-byte boundaries, the first
    // of the CTA at or before token i0
    int first = i0 - (int)(((uintptr_t)l + (size_t)i0 * ES) % 16) / ES + row.warp * (32 * kTok) + row.lane * VEC;
    auto token = [&](int j, int e) { return first + j * (32 * VEC) + e; };

    // The row that this SM takes next, into L2 while this one is worked on: one CTA
    // holds the SM's registers, so nothing else overlaps its loads with arithmetic.
    if (CL == 1 && threadIdx.x == 0 && r + a.ahead < a.rows) {
        const uintptr_t n0 = (uintptr_t)l + (size_t)a.ahead * a.ld * ES, n1 = n0 + (size_t)V * ES;
        const uintptr_t p0 = (n0 + 15) & ~(uintptr_t)15, p1 = n1 & ~(uintptr_t)15;
        if (p1 > p0)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p0), "r"((uint32_t)(p1 - p0)) : "memory");
    }
    uint32_t w[kTok];   // logits, then weights
    const int w0 = token(0, 0) - row.lane * VEC;   // this warp's tokens
    if (w0 >= i0 && w0 + 32 * kTok <= i1) {
        uint4 q[J];   // all loads in flight at once
#pragma unroll
        for (int j = 0; j < J; j++) q[j] = *reinterpret_cast<const uint4*>(l + (size_t)token(j, 0) * ES);
#pragma unroll
        for (int j = 0; j < J; j++) {
            const uint32_t qw[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                if constexpr (DT == FL_F32) w[j * VEC + e] = qw[e];
                else if constexpr (DT == FL_F16) {
                    const __half2 h = *reinterpret_cast<const __half2*>(&qw[e >> 1]);
                    w[j * VEC + e] = __float_as_uint((e & 1) ? __high2float(h) : __low2float(h));
                } else w[j * VEC + e] = (e & 1) ? qw[e >> 1] & 0xffff0000u : qw[e >> 1] << 16;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kTok; i++) {
            const int t = token(i / VEC, i % VEC);
            w[i] = __float_as_uint(t >= i0 && t < i1 ? logit<DT>(l, t) : -INFINITY);
        }
    }
    float mx = -INFINITY;   // NaN is never the larger
#pragma unroll
    for (int i = 0; i < kTok; i++) mx = fmaxf(mx, __uint_as_float(w[i]));
    row.started();
    mx = unsortable(row.max32(sortable(mx)));
    if (mx == INFINITY) {
        mx = FLT_MAX;
#pragma unroll
        for (int i = 0; i < kTok; i++) w[i] = __float_as_uint(canon(__uint_as_float(w[i])));
    }
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    if (mx == -INFINITY || !(T > 0.0f)) {
        uint32_t best = 0;   // complement of the lowest index with the largest logit
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (__uint_as_float(w[j * VEC + e]) == mx && token(j, e) >= i0 && token(j, e) < i1)
                    best = max(best, ~(uint32_t)token(j, e));
        best = row.max32(best);
        if (row.rank == 0 && threadIdx.x == 0) a.tokens[r] = mx == -INFINITY ? -1 : (int)~best;
        return;
    }
    // The first token, in order, at which the running sum of the values that
    // f(sum, i, token, t) adds exceeds target(total); the values may carry the
    // tag. to_all: the index goes to every thread.
    auto locate = [&](uint32_t t, auto f, auto target, bool to_all) __attribute__((always_inline)) -> uint32_t {
        uint32_t own = 0;
#pragma unroll
        for (int j = 0; j < J; j++) {
            uint32_t g = 0;
#pragma unroll
            for (int e = 0; e < VEC; e++) f(g, j * VEC + e, token(j, e), t);
            own += g & (kTag - 1u);
        }
        const u64* s = row.share(warp_pack(0, own));
        u64 tot = 0, c = 0, mine = 0;
#pragma unroll
        for (int i = 0; i < R::NS; i++) {
            tot += s[i];
            c += i < row.me ? s[i] : 0;
            mine = i == row.me ? s[i] : mine;
        }
        const u64 tgt = target(tot);
        uint32_t res = 0;   // complement of the index
        again(t);
        if (c <= tgt && tgt < c + mine) {   // this warp's piece: group by group
            bool found = false;
#pragma unroll
            for (int j = 0; j < J; j++) {
                uint32_t v[VEC], g = 0;
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    v[e] = 0;
                    f(v[e], j * VEC + e, token(j, e), t);
                    v[e] &= kTag - 1u;
                    g += v[e];
                }
                const u64 all_g = warp_pack(0, g);
                if (!found && tgt < c + all_g) {
                    found = true;
                    u64 run = g;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const u64 y = __shfl_up_sync(0xffffffffu, run, o);
                        if (row.lane >= o) run += y;
                    }
                    u64 b = c + run - g;
                    if (b <= tgt && tgt < b + g) {
#pragma unroll
                        for (int e = 0; e < VEC; e++) {
                            if (res == 0 && tgt < b + v[e]) res = ~(uint32_t)token(j, e);
                            b += v[e];
                        }
                    }
                }
                c += all_g;
            }
        }
        if (to_all) return ~row.max32(res);
        if (res) a.tokens[r] = (int)~res;
        return 0u;
    };

    int k = a.top_k ? a.top_k[r] : 0;
    uint32_t lo;   // kept: the weights >= lo
    // Once, and once more without top-k where its cut lies among weights that are not
    // ordered as their logits are (kUnorderedMin)
    for (;;) {
        // x / T rounded to nearest from one reciprocal (Markstein: with r the
        // rounded 1 / T, q = x r corrected by r (x - q T) is the rounded quotient
        // unless T's fraction is all ones), where neither it nor a quotient that
        // gives a weight leaves the normal range; quotients beyond -17 give 0
        const uint32_t tb = __float_as_uint(T);
        if (T > 1e-20f && T < 1e20f && (tb & 0x7fffffu) != 0x7fffffu) {
            const float rt = __frcp_rn(T), low = -18.0f * T;
#pragma unroll
            for (int i = 0; i < kTok; i++) {
                const float x = __fsub_rn(__uint_as_float(w[i]), mx);
                const float xc = fmaxf(x, low);   // its weight is 0 too, and its quotient in range
                const float q0 = __fmul_rn(xc, rt);
                w[i] = sample_weight(__fmaf_rn(__fmaf_rn(-q0, T, xc), rt, q0)) + kTag;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kTok; i++) w[i] = sample_weight(__fdiv_rn(__fsub_rn(__uint_as_float(w[i]), mx), T)) + kTag;
        }
        const u64 all = at_least(row, w, 1u);
        u64 slo = all, shi = 0;
        lo = 1u;
        u64 z = all & kMass;
        u64 ties = 0, room = 0;    // weights equal to lo, and how many of them top-k keeps
        bool apart = false;        // ties are those of lo - 1 and lo + 1, too
        if (k > 0 && (u64)k < (all >> kMassBits)) {
            lo = bisect(row, w, 1u, kOne + 1u, slo, shi, [&](u64 s) { return (s >> kMassBits) >= (u64)k; });
            ties = (slo - shi) >> kMassBits;
            room = (u64)k - (shi >> kMassBits);
            z = (shi & kMass) + room * lo;
            if (lo >= kUnorderedMin && lo <= kUnorderedMax) {
                const uint32_t from = lo - 1u + kTag;
                uint32_t c = 0;
#pragma unroll
                for (int i = 0; i < kTok; i++) c += w[i] - from <= 2u;
                const u64 n = row.sum(0, c);
                apart = n != ties;
                if (apart) {
                    room = (u64)k - (at_least(row, w, lo + 2u) >> kMassBits);
                    ties = n;
                }
            }
        }
        const uint32_t kth = ties > room ? lo : 0u;   // the weight of which only some are kept
        const float tp = a.top_p ? a.top_p[r] : 1.0f;
        if (tp < 1.0f && !apart) {
            const u64 need = (u64)(((u128)max(1u, fixed24(tp)) * z + (kOne - 1u)) >> 24);
            auto ok = [&](u64 s) { return (s & kMass) >= need; };
            // after top-k within the weights above the k-th, which are all kept, if they suffice
            if (ties == 0 || ok(shi)) {
                if (ties) slo = shi;
                shi = 0;
                lo = bisect(row, w, ties ? lo + 1u : 1u, kOne + 1u, slo, shi, ok);
            }
        }
        if (a.min_p && !apart) lo = max(lo, fixed24(a.min_p[r]));

        if (apart || (kth && lo == kth)) {
            // top-k keeps `room` of the `ties` weights equal to lo (or next to it): the
            // largest logits, equal ones in index order (different logits can share a
            // weight, far below the maximum thousands of them)
            constexpr uint32_t kHalf = 0x80000000u, kKept = 1u << 29;
            const uint32_t tie = lo + kTag, from = tie - (apart ? 1u : 0u), span = apart ? 2u : 0u;
            asm volatile("" : "+r"(first));   // nothing of the 64 addresses is kept from before
            uint32_t top, bot;
            auto range = [&]() {   // of the ties' keys
                uint32_t hi = 0, lo_c = 0;
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int e = 0; e < VEC; e++)
                        if (w[j * VEC + e] - from <= span) {
                            const uint32_t s = sortable(logit<DT>(l, token(j, e)));
                            hi = max(hi, s);
                            lo_c = max(lo_c, ~s);
                        }
                top = row.max32(hi);
                bot = ~row.max32(lo_c);
            };
            range();
            u64 left = ties, need = room;
            if (top - bot >= kHalf) {   // both signs, a vast temperature: the one that the cut lies in
                uint32_t c = 0;
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int e = 0; e < VEC; e++)
                        if (w[j * VEC + e] - from <= span) c += sortable(logit<DT>(l, token(j, e))) >= kHalf;
                const u64 pos = row.sum(0, c);
                const bool up = pos >= need;
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int e = 0; e < VEC; e++)
                        if (w[j * VEC + e] - from <= span && (sortable(logit<DT>(l, token(j, e))) >= kHalf) != up)
                            w[j * VEC + e] = up ? kTag : w[j * VEC + e] | kKept;   // dropped, or kept without more ado
                left = up ? pos : left - pos;
                need = up ? need : need - pos;
                range();
            }
            if (need < left) {
                // the ties as their keys less the smallest, below 2^31, marked by the top bit
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int e = 0; e < VEC; e++)
                        if (w[j * VEC + e] - from <= span)
                            w[j * VEC + e] = kHalf + (sortable(logit<DT>(l, token(j, e))) - bot);
                // cut: as many keys at or above it as are needed, or the largest with at least as many
                uint32_t cut = kHalf, end = kHalf + (top - bot) + 1u;
                u64 at_cut = left, at_end = 0;
                while (end - cut > 1u && at_cut != need) {
                    const uint32_t mid = cut + (end - cut) / 2u;
                    uint32_t c = 0;
#pragma unroll
                    for (int i = 0; i < kTok; i++) c += w[i] >= mid;
                    const u64 n = row.sum(0, c);
                    if (n >= need) { cut = mid; at_cut = n; } else { end = mid; at_end = n; }
                }
                uint32_t last = 0xffffffffu;   // of the tokens at the cut, the last one kept
                if (at_cut != need)
                    last = locate(cut, [&](uint32_t& sum, int i, int, uint32_t t) { sum += w[i] == t; },
                                  [&](u64) { return need - at_end - 1; }, true);
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const uint32_t x = w[j * VEC + e];
                        if (x >= kHalf)
                            w[j * VEC + e] = x > cut || (x == cut && (uint32_t)token(j, e) <= last) ? tie : kTag;
                    }
            }
#pragma unroll
            for (int i = 0; i < kTok; i++) w[i] &= ~kKept;
            if (apart) {   // the logits that top-k keeps; the other rules on them alone
                asm volatile("" : "+r"(first));
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int e = 0; e < VEC; e++)
                        w[j * VEC + e] =
                            __float_as_uint(w[j * VEC + e] >= from ? logit<DT>(l, token(j, e)) : -INFINITY);
                k = 0;
                continue;
            }
        }
        break;
    }
    const uint32_t U = min(fixed24(a.u[r]), kOne - 1u);
    locate(lo + kTag, [&](uint32_t& sum, int i, int, uint32_t t) { add_if_ge(sum, w[i], t, row.one); },
           [&](u64 total) { return (u64)(((u128)U * total) >> 24); }, false);
}

template <int DT, int NT, int CL>
cudaError_t launch_sample(const SampleArgs& a, int rows, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CL;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(rows * CL);
    cfg.blockDim = dim3(NT);
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = CL > 1;
    return cudaLaunchKernelEx(&cfg, sample_rows_kernel<DT, NT, CL>, a);
}

// Tokens a CTA holds: its first group may begin up to 7 tokens early.
constexpr int cta_tokens(int threads) { return threads * kTok - 8; }
constexpr int kMaxVocab = 262000;   // eight CTAs of 512 threads

int sample_sms() {
    static const int sms = [] {
        int dev = 0, n = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        return n > 0 ? n : 148;
    }();
    return sms;
}

template <int DT>
cudaError_t sample_dt(SampleArgs a, int rows, cudaStream_t s) {
    // a cluster of cl CTAs of `threads` that covers a row
    auto fits = [&](int threads, int cl) {
        a.seg = ((a.V + cl - 1) / cl + 7) / 8 * 8;
        return a.seg <= cta_tokens(threads);
    };
    a.ahead = 4 * sample_sms();
    if (fits(128, 1)) return launch_sample<DT, 128, 1>(a, rows, s);
    // while all CTAs of four to a row are resident (several share an SM): one row of
    // 32064 took 17 us in four CTAs of 128 threads, 20 in one of 512
    if (rows * 4 <= sample_sms() * 2 && fits(128, 4)) return launch_sample<DT, 128, 4>(a, rows, s);
    a.ahead = sample_sms();
    if (fits(512, 1)) return launch_sample<DT, 512, 1>(a, rows, s);
    if (fits(256, 8)) return launch_sample<DT, 256, 8>(a, rows, s);
    if (fits(512, 8)) return launch_sample<DT, 512, 8>(a, rows, s);
    return cudaErrorInvalidValue;
}

}  // namespace

}  // namespace fl

using namespace fl;

FL_API int fl_cuda_sample(const void* logits, int dtype, size_t ld, int rows, int V, const float* temperature,
                          const int* top_k, const float* top_p, const float* min_p, const float* u, int* tokens,
                          void* stream) {
    if (rows < 0 || rows > (1 << 24) || V < 1) return set_error(FL_E_INVAL, "sample: bad sizes");
    if (dtype != FL_F32 && dtype != FL_F16 && dtype != FL_BF16)
        return set_error(FL_E_INVAL, "sample: dtype must be FL_F32, FL_F16 or FL_BF16");
    if (rows == 0) return FL_OK;
    if (!logits || !u || !tokens) return set_error(FL_E_INVAL, "sample: NULL argument");
    if (V > kMaxVocab) return set_error(FL_E_UNSUPPORTED, "sample: at most 262000 tokens");
    if (rows > 1 && ld < (size_t)V) return set_error(FL_E_INVAL, "sample: the row stride is below V");
    if ((uintptr_t)logits % (dtype == FL_F32 ? 4 : 2))
        return set_error(FL_E_INVAL, "sample: logits are not aligned to their type");
    const struct {
        const void* p;
        const char* name;
    } arrays[] = {{temperature, "sample: temperature"}, {top_k, "sample: top_k"}, {top_p, "sample: top_p"},
                  {min_p, "sample: min_p"},             {u, "sample: u"},         {tokens, "sample: tokens"}};
    for (const auto& x : arrays)
        if ((uintptr_t)x.p % 4) return set_error(FL_E_INVAL, std::string(x.name) + " is not aligned to its type");
    FL_CHECK(check_device_ptr(logits, "sample: logits"));
    for (const auto& x : arrays)
        if (x.p) FL_CHECK(check_device_ptr(x.p, x.name));
    cudaStream_t s = stream ? (cudaStream_t)stream : device_stream();
    const SampleArgs a = {logits, ld, V, 0, rows, 0, temperature, top_p, min_p, u, top_k, tokens};
    FL_CHECK_CUDA(dtype == FL_F32 ? sample_dt<FL_F32>(a, rows, s)
                                  : dtype == FL_F16 ? sample_dt<FL_F16>(a, rows, s) : sample_dt<FL_BF16>(a, rows, s));
    return FL_OK;
}
