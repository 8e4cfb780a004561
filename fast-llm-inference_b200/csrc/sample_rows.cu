// One token per logits row from given uniform numbers (sm_100a): temperature,
// top-k, min-p and top-p on the integer weights of the library's sampling rule
// (fl_sample.cuh), so every sum is exact and the draw does not depend on the
// order of any reduction. The rule is stated at fl_cuda_sample in
// include/fl_cuda.h.
//
// A row is held by one CTA, or by a cluster of up to eight: every thread reads
// 32 tokens at most, once, turns them into weights and keeps those in
// registers. A threshold (of top-k by count, of top-p by mass) is found by
// bisection between weights lo and hi, at their geometric mean while they lie
// apart: after a few passes over the registers the undecided weights fit a
// list in shared memory, and the remaining passes touch one or two of them per
// thread. Counts and masses share one 64-bit word (44 bits of mass, V < 2^20),
// and a pass costs one barrier. The draw is a two-level prefix sum in token
// order: warps' sums, then the lanes of the warp that the target falls into.
// Bound by instructions: about 25 a token for its weight, 3 for each pass.
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
constexpr int kTok = 32;          // tokens per thread
constexpr int kList = 2048;       // undecided weights of a CTA in shared memory
constexpr int kMassBits = 44;
constexpr u64 kMass = (1ull << kMassBits) - 1;

struct SampleArgs {
    const void* logits;
    size_t ld;
    int V, seg;                   // tokens of a CTA of the row's cluster
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* tokens;
};

// A logit as the rule reads it: NaN counts as -inf, +inf as the largest float, -0 as 0.
__device__ __forceinline__ float canon(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX) + 0.0f; }
template <int DT>
__device__ __forceinline__ float logit(const void* l, int i) {
    if constexpr (DT == FL_F32) return canon(static_cast<const float*>(l)[i]);
    else if constexpr (DT == FL_F16) return canon(__half2float(static_cast<const __half*>(l)[i]));
    else return canon(__bfloat162float(static_cast<const __nv_bfloat16*>(l)[i]));
}
// Orders floats as unsigned integers.
__device__ __forceinline__ uint32_t sortable(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unsortable(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
// trunc(p 2^24) within [0, 2^24]; 0 for NaN.
__device__ __forceinline__ uint32_t fixed24(float p) {
    return __float2uint_rz(__fmul_rn(fminf(fmaxf(p, 0.0f), 1.0f), 16777216.0f));
}

// Sum over the warp modulo 2^64, from three integer reductions of the word's parts.
__device__ __forceinline__ u64 warp_sum64(u64 v) {
    const uint32_t a = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0xffffffu);
    const uint32_t b = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 24) & 0xffffffu);
    const uint32_t c = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 48));
    return (u64)a + ((u64)b << 24) + ((u64)c << 48);
}

// Reductions and prefix sums over the threads of a row's CTA or cluster.
template <int NT, int CL>
struct Row {
    static constexpr int NW = NT / 32;
    struct Shared {
        u64 slot[2][CL * NW];
        u64 cell[kTok * NW];
        uint32_t list[kList];
        int nlist, found;
    };
    Shared& sm;
    int lane, warp, rank;
    int phase = 0;

    __device__ Row(Shared& s) : sm(s), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), rank(0) {
        if (CL > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    }
    __device__ __forceinline__ void sync() {
        if constexpr (CL > 1)
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else
            __syncthreads();
    }
    // lane 0 of every warp: v into this warp's slot of every CTA of the cluster
    __device__ __forceinline__ void push(u64 v) {
        u64* p = &sm.slot[phase][rank * NW + warp];
        if constexpr (CL > 1) {
            const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
            if (lane < CL) {
                uint32_t ra;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(a), "r"(lane));
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(ra), "l"(v) : "memory");
            }
        } else if (lane == 0) {
            *p = v;
        }
    }
    // Two slot sets in turn: a thread that is a pass ahead writes the other one.
    __device__ __forceinline__ u64 sum(u64 v) {
        push(warp_sum64(v));
        sync();
        u64 t = 0;
#pragma unroll
        for (int i = 0; i < CL * NW; i += 32)
            if (i + lane < CL * NW) t += sm.slot[phase][i + lane];
        phase ^= 1;
        return warp_sum64(t);
    }
    __device__ __forceinline__ uint32_t max32(uint32_t v) {
        push(__reduce_max_sync(0xffffffffu, v));
        sync();
        u64 t = 0;
#pragma unroll
        for (int i = 0; i < CL * NW; i += 32)
            if (i + lane < CL * NW) t = max(t, sm.slot[phase][i + lane]);
        phase ^= 1;
        return __reduce_max_sync(0xffffffffu, (uint32_t)t);
    }
};

// (count, mass) of the weights at or above t among the thread's registers.
__device__ __forceinline__ u64 at_least(const uint32_t (&w)[kTok], uint32_t t) {
    uint32_t m = 0, c = 0;   // 32 weights of at most 2^24 sum below 2^30
#pragma unroll
    for (int i = 0; i < kTok; i++) {
        m += w[i] >= t ? w[i] : 0u;
        c += w[i] >= t;
    }
    return ((u64)c << kMassBits) + m;
}

// The largest t in [lo, hi) with ok(sum of the weights >= t), given that
// ok holds at lo and not at hi; slo and shi are those sums, and on return the
// ones at t and t + 1.
template <class R, class Ok>
__device__ __forceinline__ uint32_t bisect(R& row, const uint32_t (&w)[kTok], uint32_t lo, uint32_t hi, u64& slo,
                                           u64& shi, Ok ok) {
    auto middle = [&]() -> uint32_t {
        if (hi >> 1 > lo) {
            const uint32_t g = __float2uint_rz(sqrtf(__uint2float_rz(lo)) * sqrtf(__uint2float_rz(hi)));
            return min(max(g, lo + 1), hi - 1);
        }
        return lo + (hi - lo) / 2u;
    };
    while (hi - lo > 1u && ((slo - shi) >> kMassBits) > kList) {
        const uint32_t mid = middle();
        const u64 s = row.sum(at_least(w, mid));
        if (ok(s)) { lo = mid; slo = s; } else { hi = mid; shi = s; }
    }
    if (hi - lo <= 1u) return lo;
    // the undecided weights of this CTA as a list
    if (threadIdx.x == 0) row.sm.nlist = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTok; i++)
        if (w[i] >= lo && w[i] < hi) row.sm.list[atomicAdd(&row.sm.nlist, 1)] = w[i];
    __syncthreads();
    constexpr int PT = (kList + R::NW * 32 - 1) / (R::NW * 32);
    const int n = row.sm.nlist;
    uint32_t q[PT];
#pragma unroll
    for (int i = 0; i < PT; i++) {
        const int at = threadIdx.x + i * R::NW * 32;
        q[i] = at < n ? row.sm.list[at] : 0u;
    }
    const u64 base = shi;
    while (hi - lo > 1u) {
        const uint32_t mid = middle();
        uint32_t m = 0, c = 0;
#pragma unroll
        for (int i = 0; i < PT; i++) {
            const bool in = q[i] >= mid;
            m += in ? q[i] : 0u;
            c += in;
        }
        const u64 s = base + row.sum(((u64)c << kMassBits) + m);
        if (ok(s)) { lo = mid; slo = s; } else { hi = mid; shi = s; }
    }
    return lo;
}

template <int DT, int NT, int CL>
__global__ void __launch_bounds__(NT) sample_rows_kernel(const SampleArgs a) {
    typedef Row<NT, CL> R;
    constexpr int ES = DT == FL_F32 ? 4 : 2, VEC = 16 / ES, J = kTok / VEC;
    __shared__ typename R::Shared shared;
    R row(shared);
    const int r = blockIdx.x / CL;
    const char* l = static_cast<const char*>(a.logits) + (size_t)r * a.ld * ES;
    const int i0 = row.rank * a.seg, i1 = min(a.V, i0 + a.seg);   // this CTA's tokens
    // token of (group j, element e) of this thread: its groups of VEC tokens
    // begin on 16-byte boundaries, the first at or before token i0
    const int first = i0 - (int)(((uintptr_t)l + (size_t)i0 * ES) % 16) / ES + (int)threadIdx.x * VEC;
    auto token = [&](int j, int e) { return first + j * (NT * VEC) + e; };

    uint32_t w[kTok];   // logits as sortable keys, then weights
    uint32_t kmax = 0;
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int t0 = token(j, 0);
        if (t0 >= i0 && t0 + VEC <= i1) {
            const uint4 q = *reinterpret_cast<const uint4*>(l + (size_t)t0 * ES);
            const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                float x;
                if constexpr (DT == FL_F32) x = __uint_as_float(qw[e]);
                else if constexpr (DT == FL_F16) {
                    const __half2 h = *reinterpret_cast<const __half2*>(&qw[e >> 1]);
                    x = (e & 1) ? __high2float(h) : __low2float(h);
                } else x = __uint_as_float((e & 1) ? qw[e >> 1] & 0xffff0000u : qw[e >> 1] << 16);
                w[j * VEC + e] = sortable(canon(x));
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const int t = t0 + e;
                w[j * VEC + e] = sortable(t >= i0 && t < i1 ? logit<DT>(l, t) : -INFINITY);
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) kmax = max(kmax, w[j * VEC + e]);
    }
    kmax = row.max32(kmax);
    const float mx = unsortable(kmax);
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    if (mx == -INFINITY || !(T > 0.0f)) {
        uint32_t best = 0;   // complement of the lowest index with the largest logit
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (w[j * VEC + e] == kmax && token(j, e) >= i0 && token(j, e) < i1)
                    best = max(best, ~(uint32_t)token(j, e));
        best = row.max32(best);
        if (row.rank == 0 && threadIdx.x == 0) a.tokens[r] = mx == -INFINITY ? -1 : (int)~best;
        return;
    }
    // x / T rounded to nearest from one reciprocal (Markstein: with r the
    // rounded 1 / T, q = x r corrected by r (x - q T) is the rounded quotient
    // unless T's fraction is all ones), where neither it nor a quotient that
    // gives a weight leaves the normal range; quotients beyond -17 give 0
    const uint32_t tb = __float_as_uint(T);
    if (T > 1e-20f && T < 1e20f && (tb & 0x7fffffu) != 0x7fffffu) {
        const float rt = __frcp_rn(T), low = -18.0f * T;
#pragma unroll
        for (int i = 0; i < kTok; i++) {
            const float x = __fsub_rn(unsortable(w[i]), mx);
            const float q0 = __fmul_rn(x, rt);
            const float q = __fmaf_rn(__fmaf_rn(-q0, T, x), rt, q0);
            w[i] = x > low ? sample_weight(q) : 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kTok; i++) w[i] = sample_weight(__fdiv_rn(__fsub_rn(unsortable(w[i]), mx), T));
    }
    const u64 all = row.sum(at_least(w, 1u));
    u64 slo = all, shi = 0;
    uint32_t lo = 1u;          // kept: the weights >= lo
    u64 z = all & kMass;
    const int k = a.top_k ? a.top_k[r] : 0;
    u64 ties = 0, room = 0;    // weights equal to lo, and how many of them top-k keeps
    if (k > 0 && (u64)k < (all >> kMassBits)) {
        lo = bisect(row, w, 1u, kOne + 1u, slo, shi, [&](u64 s) { return (s >> kMassBits) >= (u64)k; });
        ties = (slo - shi) >> kMassBits;
        room = (u64)k - (shi >> kMassBits);
        z = (shi & kMass) + room * lo;
    }
    const uint32_t kth = ties > room ? lo : 0u;   // the weight of which only some are kept
    const float tp = a.top_p ? a.top_p[r] : 1.0f;
    if (tp < 1.0f) {
        const u128 need = (u128)max(1u, fixed24(tp)) * z;
        auto ok = [&](u64 s) { return ((u128)(s & kMass) << 24) >= need; };
        // after top-k within the weights above the k-th, which are all kept, if they suffice
        if (ties == 0 || ok(shi)) {
            if (ties) slo = shi;
            shi = 0;
            lo = bisect(row, w, ties ? lo + 1u : 1u, kOne + 1u, slo, shi, ok);
        }
    }
    if (a.min_p) lo = max(lo, fixed24(a.min_p[r]));

    // The first token, in order, at which the running sum of f(i, token)
    // exceeds target(total); to_all: the index goes to every thread.
    auto locate = [&](auto f, auto target, bool to_all) __attribute__((always_inline)) -> uint32_t {
        u64 own = 0;
#pragma unroll
        for (int j = 0; j < J; j++) {
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < VEC; e++) c += f(j * VEC + e, token(j, e));
            const u64 s = warp_sum64(c);
            if (row.lane == 0) shared.cell[j * R::NW + row.warp] = s;
            own += c;
        }
        // total, and the sum of the CTAs before this one
        row.push(warp_sum64(own));
        if (CL == 1) row.sync(); else { __syncthreads(); row.sync(); }
        u64 tot = 0, before = 0;
#pragma unroll
        for (int i = 0; i < CL * R::NW; i += 32)
            if (i + row.lane < CL * R::NW) {
                const u64 s = shared.slot[row.phase][i + row.lane];
                tot += s;
                before += i + row.lane < row.rank * R::NW ? s : 0;
            }
        row.phase ^= 1;
        tot = warp_sum64(tot);
        before = warp_sum64(before);
        const u64 tgt = target(tot);
        // the cell: lane n takes the cells [n PC, (n + 1) PC)
        constexpr int CELLS = J * R::NW, PC = (CELLS + 31) / 32;
        u64 inc = 0;
#pragma unroll
        for (int i = 0; i < PC; i++) inc += row.lane * PC + i < CELLS ? shared.cell[row.lane * PC + i] : 0;
        const u64 mine = inc;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
            if (row.lane >= o) inc += y;
        }
        u64 c = before + inc - mine;
        int cell = -1;
        for (int i = 0; i < PC; i++) {
            const u64 s = row.lane * PC + i < CELLS ? shared.cell[row.lane * PC + i] : 0;
            if (cell < 0) {
                if (c <= tgt && tgt < c + s) cell = row.lane * PC + i;
                else c += s;
            }
        }
        const uint32_t who = __ballot_sync(0xffffffffu, cell >= 0);
        uint32_t res = 0;   // complement of the index
        if (who) {
            const int src = __ffs(who) - 1;
            cell = __shfl_sync(0xffffffffu, cell, src);
            c = __shfl_sync(0xffffffffu, c, src);
            if (cell % R::NW == row.warp) {
                uint32_t f4[VEC] = {}, sum = 0;
                int t0 = 0;
#pragma unroll
                for (int j = 0; j < J; j++) {   // selects: an index of run time would move w to local memory
                    const bool here = j == cell / R::NW;
                    t0 = here ? token(j, 0) : t0;
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const uint32_t v = f(j * VEC + e, token(j, e));
                        f4[e] = here ? v : f4[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < VEC; e++) sum += f4[e];
                u64 run = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 y = __shfl_up_sync(0xffffffffu, run, o);
                    if (row.lane >= o) run += y;
                }
                u64 b = c + run - sum;
                if (b <= tgt && tgt < b + sum) {
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        if (res == 0 && tgt < b + f4[e]) res = ~(uint32_t)(t0 + e);
                        b += f4[e];
                    }
                }
            }
        }
        if (to_all) return ~row.max32(res);
        if (res) a.tokens[r] = (int)~res;
        return 0u;
    };

    if (kth && lo == kth) {
        // top-k keeps `room` of the `ties` weights equal to kth: the largest
        // logits, equal ones in index order (different logits can share a weight)
        uint32_t top = 0, bot = 0;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (w[j * VEC + e] == kth) {
                    const uint32_t s = sortable(logit<DT>(l, token(j, e)));
                    top = max(top, s);
                    bot = max(bot, ~s);
                }
        top = row.max32(top);
        bot = ~row.max32(bot);
        auto key_count = [&](uint32_t t) {   // ties with a key of at least t
            u64 c = 0;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    if (w[j * VEC + e] == kth) c += sortable(logit<DT>(l, token(j, e))) >= t;
            return row.sum(c);
        };
        // bot: the largest key with `room` ties at or above it
        uint32_t up = top + 1u;
        u64 above = 0;
        while (up - bot > 1u) {
            const uint32_t mid = bot + (up - bot) / 2u;
            const u64 c = key_count(mid);
            if (c >= room) bot = mid; else { up = mid; above = c; }
        }
        auto equal = [&](int i, int t) -> uint32_t { return w[i] == kth && sortable(logit<DT>(l, t)) == bot; };
        const uint32_t last = locate(equal, [&](u64) { return room - above - 1; }, true);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (w[j * VEC + e] == kth) {
                    const uint32_t s = sortable(logit<DT>(l, token(j, e)));
                    if (s < bot || (s == bot && (uint32_t)token(j, e) > last)) w[j * VEC + e] = 0u;
                }
    }
    const uint32_t U = min(fixed24(a.u[r]), kOne - 1u);
    locate([&](int i, int) -> uint32_t { return w[i] >= lo ? w[i] : 0u; },
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
constexpr int kSmall = 256, kLarge = 1024;
constexpr int cta_tokens(int threads) { return threads * kTok - 8; }
constexpr int kMaxVocab = 262000;   // eight CTAs

template <int DT>
cudaError_t sample_dt(SampleArgs a, int rows, cudaStream_t s) {
    const int V = a.V;
    auto seg = [&](int cl) { return ((V + cl - 1) / cl + 7) / 8 * 8; };
    int cl = 1;
    if (V <= cta_tokens(kSmall)) {
        a.seg = seg(1);
        return launch_sample<DT, kSmall, 1>(a, rows, s);
    }
    while (seg(cl) > cta_tokens(kLarge)) cl *= 2;
    a.seg = seg(cl);
    switch (cl) {
        case 1: return launch_sample<DT, kLarge, 1>(a, rows, s);
        case 2: return launch_sample<DT, kLarge, 2>(a, rows, s);
        case 4: return launch_sample<DT, kLarge, 4>(a, rows, s);
        default: return launch_sample<DT, kLarge, 8>(a, rows, s);
    }
}

}  // namespace

}  // namespace fl

using namespace fl;

FL_API int fl_cuda_sample(const void* logits, int dtype, size_t ld, int rows, int V, const float* temperature,
                          const int* top_k, const float* top_p, const float* min_p, const float* u, int* tokens,
                          void* stream) {
    if (rows < 0 || V < 1) return set_error(FL_E_INVAL, "sample: bad sizes");
    if (dtype != FL_F32 && dtype != FL_F16 && dtype != FL_BF16)
        return set_error(FL_E_INVAL, "sample: dtype must be FL_F32, FL_F16 or FL_BF16");
    if (rows == 0) return FL_OK;
    if (!logits || !u || !tokens) return set_error(FL_E_INVAL, "sample: NULL argument");
    if (V > kMaxVocab) return set_error(FL_E_UNSUPPORTED, "sample: at most 262000 tokens");
    if (rows > 1 && ld < (size_t)V) return set_error(FL_E_INVAL, "sample: the row stride is below V");
    if ((uintptr_t)logits % (dtype == FL_F32 ? 4 : 2))
        return set_error(FL_E_INVAL, "sample: logits are not aligned to their type");
    FL_CHECK(ensure_device());
    cudaStream_t s = stream ? (cudaStream_t)stream : device_stream();
    const SampleArgs a = {logits, ld, V, 0, temperature, top_p, min_p, u, top_k, tokens};
    FL_CHECK_CUDA(dtype == FL_F32 ? sample_dt<FL_F32>(a, rows, s)
                                  : dtype == FL_F16 ? sample_dt<FL_F16>(a, rows, s) : sample_dt<FL_BF16>(a, rows, s));
    return FL_OK;
}
