// Attention of many query rows over the paged 8-bit KV cache (prompt chunks,
// draft trees of grouped heads) on the 5th-generation tensor cores, sm_100a.
// The mathematics is that of kv8_attn.cu.
//
// A CTA takes two tiles of 128 packed query rows of one kv head at a time,
// against pages of 64 keys: S = Q K^T (128 x 64) and O += P V (128 x head_dim), all
// tcgen05.mma.kind::f16, K, V and Q in shared memory (SWIZZLE_128B, K-major), P in
// TMEM, accumulators in TMEM: per tile two S buffers of 64 columns and O, 512
// columns in all.
//  - warps 0-3 and 4-7: softmax of either tile, one query row a thread. They write
//    Q at first, then per page read S (tcgen05.ld), keep the running reference and
//    sum, and write P as halves over S (from shared memory, whose bandwidth bounds
//    the products, P would be written and read once more). The reference follows the
//    maximum only once it lags by 2^8, so O is seldom read back and rescaled.
//  - warps 8-11: conversion, one 16-position block of the page a warp. The codes
//    come as 16-byte pieces (fl_kv8.h), a page ahead of their use, and go to one of
//    two stages as halves: a K piece is two 16-byte chunks of two keys' rows; a V
//    piece holds four keys of four dimensions, so V^T is written without a
//    transposition. V is scaled by its block's scale over the accumulators' (next_vref; a power
//    of two, in the multiply-add that removes the INT8 offset). Both tiles use it.
//  - warp 12: one thread issues the products, S of the next page before P V of
//    this, tile by tile, so that one tile's softmax runs beside the other's
//    products. (Issued by a conversion warp, the two waited for each other: 1.05 ms
//    instead of the figure below.)
// f32 rows take two halves for Q and for P (22 bits): twice the products.
//
// Every product drops the bits of its sums below 2^-24, towards zero: over n products
// sums of one sign fall short by about n 2^-25. That is 1.4e-4 for f32 rows over 30 k
// keys, so their O goes to sums rounded to nearest, in the workspace, every 4 pages (32
// products, remainders first while the sums are small): f32 chunks of the sizes below
// take 0.97 ms, without 0.82. 16-bit rows have half the products and round coarser:
// they keep what is lost, about 2^-16 for each 4096 keys.
//
// Bound by the issue of the products, about 80 clocks each: 24 per page and pair of
// tiles, 2500 of some 3900 clocks; then by the softmax warps' chain per page (2700).
// Prompt chunks of 0.8 to 2 k rows behind 0 to 6 k keys (32 / 8 heads of 128, 0.34
// TFLOP) take 0.84 ms, 0.4 PFLOP/s; the row kernel takes 2.47 ms.
//
// Waits are bounded (kKv8WaitClocks, about 2 s); on expiry the CTA raises an error word,
// stops, waits (bounded) for all products that it issued, frees TMEM and exits.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "fl_common.cuh"
#include "fl_kv8.h"
#include "fl_kv8_attn.cuh"
#include "fl_kv8_types.cuh"

namespace fl {

namespace {

__device__ int g_kv8_error = 0;
std::atomic<bool> g_kv8_launched{false};   // the kernel was launched (or captured) in this process

constexpr int kRows = 128;               // query rows of a tile
constexpr int kPair = kKv8Long;          // of a CTA's two tiles
constexpr int kThreads = 13 * 32;
constexpr float kVUp = 32.0f;            // V enters as 2^5 code / largest scale: 1152 2^5, the offset, is a half

__device__ __forceinline__ uint32_t saddr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mb_init(uint64_t* b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(saddr(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void mb_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(saddr(b)) : "memory");
}
__device__ __forceinline__ bool mb_try(uint64_t* b, uint32_t par) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(saddr(b)), "r"(par)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mb_wait(uint64_t* b, uint32_t par, long long limit) {
    if (mb_try(b, par)) return true;
    const long long t0 = clock64();
    while (!mb_try(b, par))
        if (clock64() - t0 > limit) {
            atomicOr(&g_kv8_error, 1);
            return false;
        }
    return true;
}
// By a whole warp: every lane polls, so that the warp stays together (one lane
// polling for the others left it in two pieces that ran the code after it in turn:
// 3 times the time per page).
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t par, long long limit) {
    const bool ok = mb_wait(b, par, limit);
    return __all_sync(0xffffffffu, ok);
}

// The largest V scale of a page's blocks that hold positions below end.
__device__ __forceinline__ float vscale_max(const float4& v, int k0, int end) {
    float m = k0 < end ? v.x : 0.0f;
    if (k0 + kKv8Block < end) m = fmaxf(m, v.y);
    if (k0 + 2 * kKv8Block < end) m = fmaxf(m, v.z);
    if (k0 + 3 * kKv8Block < end) m = fmaxf(m, v.w);
    return m;
}

// A page's scales, loaded a page ahead of their use (and its number two ahead).
struct Scales {
    float4 k, v;
    int page;   // of the page after the loaded one
    __device__ __forceinline__ Scales(const Kv8AttnParams& p, const int* bt, int h, int n) : page(0) {
        k = v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (n > 0) page = bt[0];
        load(p, bt, h, 0, n);
    }
    __device__ __forceinline__ void load(const Kv8AttnParams& p, const int* bt, int h, int j, int n) {
        if (j >= n) return;
        const size_t at = ((size_t)page * p.kv_heads + h) * kKv8Sub;
        k = *reinterpret_cast<const float4*>(p.ks + at);
        v = *reinterpret_cast<const float4*>(p.vs + at);
        if (j + 1 < n) page = bt[j + 1];
    }
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {   // 128-byte swizzled K-major rows, 8-row groups
    uint64_t d = (uint64_t)((addr >> 4) & 0x3FFF);
    d |= (uint64_t)(16 >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// D (f32, TMEM) (+)= A (f16, 128 x 16) B (f16, N x 16)^T.
template <int N>
__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, bool acc) {
    constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
// The same with A in TMEM: a row is a lane, a column holds two consecutive values.
template <int N>
__device__ __forceinline__ void umma_f16_ta(uint32_t d, uint32_t a, uint64_t b, bool acc) {
    constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(saddr(b))
                 : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t ta, float* f) {
    uint32_t* v = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(ta));
}
__device__ __forceinline__ void tmem_ld16(uint32_t ta, float* f) {
    uint32_t* v = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(ta));
}
__device__ __forceinline__ void tmem_st16(uint32_t ta, const float* f) {
    const uint32_t* v = reinterpret_cast<const uint32_t*>(f);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(ta),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t ta, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(ta), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
// After the wait the loaded values pass through an empty statement, so that no
// use of them moves before it.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(float (&f)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+f"(f[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void sts16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void sts8(uint32_t a, uint32_t x, uint32_t y) {
    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}

// Four V codes of a word as two half pairs times r (a power of two; off = -1152 r).
template <bool E4M3>
__device__ __forceinline__ void scaled_halves(uint32_t w, __half2 r, __half2 off, uint32_t& lo, uint32_t& hi) {
    if constexpr (E4M3) {
        uint32_t a, b;
        codes_to_halves<true>(w, a, b);
        const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&a), r);
        const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&b), r);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&a), r, off);
        const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&b), r, off);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// Shared memory of a CTA, in bytes from a 1024-byte boundary.
template <int HD, bool F32>
struct Layout {
    static constexpr int kCb = (HD + 63) / 64;                 // 64-dimension column blocks
    static constexpr int kParts = F32 ? 2 : 1;                 // halves per value of Q and P
    static constexpr int kQPart = kCb * kRows * 128, kQTile = kParts * kQPart;
    static constexpr int kKStage = kCb * kPageSize * 128, kVStage = HD * 128;
    static constexpr int kQ = 0, kK = 2 * kQTile, kV = kK + 2 * kKStage;
    static constexpr int kBytes = kV + 2 * kVStage + 1024;
};

// A row's sums over the pages before the last fold: dimensions 4 d .. 4 d + 3 at d
// kPair, so that a warp's accesses are whole lines.
template <int HD>
__device__ __forceinline__ float4* fold_row(const Kv8Tiles& tl) {
    return tl.fold + (size_t)blockIdx.x * (HD / 4) * kPair + threadIdx.x;
}

// What a tile's warps and the issuing thread signal to each other. p_full is by
// buffer, as s_full: a warp may write the next page's P before a slower one has
// written this page's, and the barrier must not count its arrival for that one.
struct TileBars {
    uint64_t q_full, s_full[2], p_full[2], pv_done;
};

template <int HD, int DT, bool E4M3>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_prefill_kernel(const Kv8AttnParams p, const Kv8Tiles tl, const int vec) {
    constexpr bool F32 = DT == FL_F32;
    typedef Layout<HD, F32> L;
    constexpr int NC = HD / 32;
    constexpr int kFold = 4;   // pages, of f32 rows
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) TileBars bars[2];
    __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], drained;
    __shared__ uint32_t tmem_s;
    __shared__ int bad_s, fail_s;   // fail_s: groups of products before the CTA gives up, 0: it does not
    __shared__ Kv8Joins joins;
    __shared__ Kv8Item it;
    const uint32_t smem = (saddr(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mb_init(&bars[i].q_full, 4);
            mb_init(&bars[i].s_full[0], 1);
            mb_init(&bars[i].s_full[1], 1);
            mb_init(&bars[i].p_full[0], 4);
            mb_init(&bars[i].p_full[1], 4);
            mb_init(&bars[i].pv_done, 1);
            mb_init(&k_full[i], 4);
            mb_init(&k_empty[i], 1);
            mb_init(&v_full[i], 4);
            mb_init(&v_empty[i], 1);
        }
        mb_init(&drained, 1);
        bad_s = joins.n = 0;
        fail_s = (int)blockIdx.x == tl.fail_cta ? tl.fail_at : 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(saddr(&tmem_s)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = tmem_s;
    // pages and items before, of the CTA and of either tile: the barriers' phases run on
    uint32_t J0 = 0, jt0 = 0, jt1 = 0, items0 = 0, items1 = 0;

    for (long long x = -1;;) {
        if (warp == 0) next_item(p, tl, x, lane, it);
        __syncthreads();
        if (it.pages == 0 || bad_s) break;
        x = it.next;
        const int h = it.head, ctx = it.ctx, row0 = it.row0, nb = it.nb;
        const int np = min(kPair, nb * p.group - it.tile * kPair);
        const int nt = np > kRows ? 2 : 1;                   // tiles with rows
        const int tok_last = (it.tile * kPair + np - 1) / p.group;
        const int kend = p.mask ? ctx + nb : ctx + tok_last + 1;
        const int k0 = it.page0 * kPageSize;                 // first key of the range
        const int n = max(0, min(it.pages, (kend - k0 + kPageSize - 1) / kPageSize));
        const int* bt = p.t.block_table + (size_t)it.seq * p.max_pages + it.page0;

        if (warp < 4 * nt) {
            // ------------------------------------------------------- softmax
            const int tile = warp >> 2, r = threadIdx.x & (kRows - 1);
            TileBars& bar = bars[tile];
            const uint32_t jb = tile ? jt1 : jt0;
            const int pr = it.tile * kPair + threadIdx.x, tok = pr / p.group;
            const int head = h * p.group + pr - tok * p.group, row = row0 + tok;
            const bool live = threadIdx.x < np && row < p.rows;
            const size_t qat = (size_t)row * p.ldq + (size_t)head * HD;
            float amax = 0.0f;
            if (live) {
#pragma unroll 4
                for (int c = 0; c < HD / 4; c++) {
                    float f[4];
                    load4<DT>(p.q, qat + 4 * c, vec, f);
#pragma unroll
                    for (int j = 0; j < 4; j++) amax = fmaxf(amax, fabsf(f[j]));
                }
            }
            // |scale| goes to the scores, its sign to the queries: factors stay positive
            const float sh = row_shift(amax);
            const float unshift = pow2_inv(sh) * fabsf(p.scale), qs = p.scale < 0.0f ? -sh : sh;
#pragma unroll 2
            for (int c = 0; c < HD / 8; c++) {
                float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (live) load8<DT>(p.q, qat + 8 * c, vec, f);
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] *= qs;
                const uint32_t a = smem + L::kQ + tile * L::kQTile + (c >> 3) * (kRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                sts16(a, h2(f[0], f[1]), h2(f[2], f[3]), h2(f[4], f[5]), h2(f[6], f[7]));
                if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < 8; j++) f[j] -= __half2float(__float2half_rn(f[j]));
                    sts16(a + L::kQPart, h2(f[0], f[1]), h2(f[2], f[3]), h2(f[4], f[5]), h2(f[6], f[7]));
                }
            }
            proxy_fence();
            __syncwarp();
            bool ok = true;
            if (lane == 0 && n > 0) mb_arrive(&bar.q_full);
            const uint32_t tq = tmem + tile * 256 + ((uint32_t)(32 * (warp & 3)) << 16);
            float m = -INFINITY, l = 0.0f, vref = 0.0f, vtop = 0.0f;
            float mf = -INFINITY, vf = 0.0f;   // reference and scale of the rounded sums
            const int lim = ctx + (p.mask ? min(nb, p.ldm) : tok + 1);   // positions this row may see
            // dead rows read some row of the mask, to no effect
            const uint8_t* mrow = p.mask + (size_t)(live ? row : min(row0, p.rows - 1)) * p.ldm;
            Scales next(p, bt, h, n);
            for (int j = 0; j < n; j++) {
                const uint32_t J = jb + j;
                const float4 ks4 = next.k;
                const float vnew = next_vref(vref, vtop, vscale_max(next.v, k0 + j * kPageSize, ctx + nb));
                next.load(p, bt, h, j + 1, n);
                if (!warp_wait(&bar.s_full[J & 1], (J >> 1) & 1, tl.wait_clocks)) { ok = false; break; }
                tc_after();
                const uint32_t sb = tq + (J & 1) * 64;
                const float f[4] = {ks4.x * unshift, ks4.y * unshift, ks4.z * unshift, ks4.w * unshift};
                const int kb = k0 + j * kPageSize;
                const bool part = kb + kPageSize > ctx + (p.mask ? 0 : (it.tile * kPair + tile * kRows) / p.group);
                uint32_t see0 = 0xffffffffu, see1 = 0xffffffffu;   // columns of this page the row sees
                if (part) {
                    const int left = lim - kb;
                    unsigned long long b = left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1ull;
                    if (p.mask)
                        for (int i = max(0, ctx - kb); i < min(64, left); i++)
                            b &= ~((unsigned long long)(mrow[kb + i - ctx] == 0) << i);
                    see0 = (uint32_t)b;
                    see1 = (uint32_t)(b >> 32);
                }
                __syncwarp();   // the TMEM accesses below take whole warps
                // S is read twice, 32 columns at a time: all 64 do not stay in registers
                float mx = -INFINITY;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    float s[32];
                    tmem_ld32(sb + 32 * w, s);
                    tmem_wait_ld(s);
                    if (part) {
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            mx = fmaxf(mx, ((w ? see1 : see0) >> i) & 1 ? s[i] * f[2 * w + (i >> 4)] : -INFINITY);
                    } else {
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            float m0 = s[16 * b], m1 = s[16 * b + 1];
#pragma unroll
                            for (int i = 2; i < 16; i += 2) {
                                m0 = fmaxf(m0, s[16 * b + i]);
                                m1 = fmaxf(m1, s[16 * b + i + 1]);
                            }
                            mx = fmaxf(mx, fmaxf(m0, m1) * f[2 * w + b]);
                        }
                    }
                }
                const bool move = mx > m + kSlack || (m == -INFINITY && mx > m);
                if (j == 0) {
                    m = mx;
                } else if (F32 && j % kFold == 0) {
                    // O to the rounded sums, in O's units; the next product begins it anew
                    if (!warp_wait(&bar.pv_done, (J - 1) & 1, tl.wait_clocks)) { ok = false; break; }
                    tc_after();
                    const float g = mf == -INFINITY ? 0.0f : ex2(mf - m) * (vf * pow2_inv(vref));
                    float4* sum = fold_row<HD>(tl);
#pragma unroll 1
                    for (int c = 0; c < NC; c++) {   // the loads of 32 dimensions at once
                        float o[32];
                        float4 b[8];
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            b[i] = j == kFold ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldcg(sum + (8 * c + i) * kPair);
                        tmem_ld32(tq + 128 + 32 * c, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            __stcg(sum + (8 * c + i) * kPair,
                                   make_float4(__fmaf_rn(b[i].x, g, o[4 * i]), __fmaf_rn(b[i].y, g, o[4 * i + 1]),
                                               __fmaf_rn(b[i].z, g, o[4 * i + 2]), __fmaf_rn(b[i].w, g, o[4 * i + 3])));
                    }
                    mf = m;
                    vf = vref;
                    m = fmaxf(m, mx);
                    l *= mf == -INFINITY ? 0.0f : ex2(mf - m);
                } else if (__any_sync(0xffffffffu, move || vnew != vref)) {
                    const float mn = fmaxf(m, mx);
                    const float al = m == -INFINITY ? 0.0f : ex2(m - mn);
                    m = mn;
                    l *= al;
                    const float g = al * (vref * pow2_inv(vnew));
                    // O: the products of the page before have to be done
                    if (!warp_wait(&bar.pv_done, (J - 1) & 1, tl.wait_clocks)) { ok = false; break; }
                    tc_after();
#pragma unroll 1
                    for (int c = 0; c < 2 * NC; c++) {
                        float o[16];
                        tmem_ld16(tq + 128 + 16 * c, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] *= g;
                        tmem_st16(tq + 128 + 16 * c, o);
                    }
                    tmem_wait_st();
                }
                vref = vnew;
                const float mr = m == -INFINITY ? 0.0f : m - kShift;
                // P over S in TMEM, two halves a column: 16 keys at columns 0, 8, 32 and 40
                // (f32 rows: their remainders 16 columns further)
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    float s[32];
                    tmem_ld32(sb + 32 * w, s);
                    tmem_wait_ld(s);
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t hi[8], lo[F32 ? 8 : 1];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            float e0 = ex2(__fmaf_rn(s[16 * c + 2 * i], f[2 * w + c], -mr));
                            float e1 = ex2(__fmaf_rn(s[16 * c + 2 * i + 1], f[2 * w + c], -mr));
                            if (part) {
                                e0 = ((w ? see1 : see0) >> (16 * c + 2 * i)) & 1 ? e0 : 0.0f;
                                e1 = ((w ? see1 : see0) >> (16 * c + 2 * i + 1)) & 1 ? e1 : 0.0f;
                            }
                            l += e0 + e1;
                            hi[i] = h2(e0, e1);
                            if constexpr (F32) {
                                e0 -= __half2float(__float2half_rn(e0));
                                e1 -= __half2float(__float2half_rn(e1));
                                lo[i] = h2(e0, e1);
                            }
                        }
                        tmem_st8(sb + 32 * w + 8 * c, hi);
                        if constexpr (F32) tmem_st8(sb + 32 * w + 16 + 8 * c, lo);
                    }
                }
                // the page before is done with, usually long ago: no thread falls two phases
                // of pv_done behind, which its parity could not tell apart
                if (j > 0 && !warp_wait(&bar.pv_done, (J - 1) & 1, tl.wait_clocks)) { ok = false; break; }
                tmem_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) mb_arrive(&bar.p_full[J & 1]);
            }
            // the row's output: normalised, to its place or to the part's slot
            if (ok && n > 0) ok = warp_wait(&bar.pv_done, (jb + n - 1) & 1, tl.wait_clocks);
            if (!ok) {
                tmem_wait_st();   // P or O may still be on its way to TMEM
                tc_before();
                if (lane == 0) atomicOr(&bad_s, 1);
            } else {
                tc_after();
                const size_t slot = 2 * (size_t)blockIdx.x + (it.split == 0);
                const float g = l != 0.0f ? __fdiv_rn(vref * (1.0f / kVUp), l) : 0.0f;
                const bool folded = F32 && n > kFold;
                const float gf = mf == -INFINITY ? 0.0f : ex2(mf - m) * (vf * pow2_inv(vref));
                const float4* sum = fold_row<HD>(tl);
#pragma unroll 1
                for (int c = 0; c < NC; c++) {
                    float o[32];
                    __syncwarp();   // rows without an output left the stores early
                    if (n > 0) {
                        tmem_ld32(tq + 128 + 32 * c, o);
                        tmem_wait_ld(o);
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        if (folded) {
                            const float4 b = __ldcg(sum + (8 * c + i / 4) * kPair);
                            o[i] = __fmaf_rn(b.x, gf, o[i]);
                            o[i + 1] = __fmaf_rn(b.y, gf, o[i + 1]);
                            o[i + 2] = __fmaf_rn(b.z, gf, o[i + 2]);
                            o[i + 3] = __fmaf_rn(b.w, gf, o[i + 3]);
                        }
                        float v[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) v[k] = n > 0 && l != 0.0f ? o[i + k] * g : 0.0f;
                        if (it.splits > 1)
                            *reinterpret_cast<float4*>(tl.part + (slot * kPair + threadIdx.x) * HD + c * 32 + i) =
                                make_float4(v[0], v[1], v[2], v[3]);
                        else if (live)
                            store4<DT>(p.out, (size_t)row * p.ldo + (size_t)head * HD + c * 32 + i, vec, v);
                    }
                }
                if (it.splits > 1) tl.part_ml[slot * kPair + threadIdx.x] = make_float2(m, l);
                tc_before();
            }
        } else if (warp >= 8 && warp < 12) {
            // ---------------------------------------------------- conversion
            const int blk = warp - 8, t4 = lane & 3, g = lane >> 2;
            // the next page's K codes are loaded once this page's are converted, and
            // its V codes likewise; page numbers and scales a page ahead
            uint4 kq[NC], vq[NC];
            Scales next(p, bt, h, n);
            size_t off = 0;
            auto load_k = [&](int page) {
                off = ((size_t)page * p.kv_heads + h) * (kPageSize * HD) + blk * (kKv8Block * HD) + lane * 16;
#pragma unroll
                for (int c = 0; c < NC; c++) kq[c] = ld_stream16(p.k + off + c * 512);
            };
            auto load_v = [&]() {
#pragma unroll
                for (int c = 0; c < NC; c++) vq[c] = ld_stream16(p.v + off + c * 512);
            };
            // K rows: key 16 blk + 4 (g / 2) + (g & 1) + 2 half, dimensions 32 c + 8 t4 .. + 7
            auto write_k = [&](uint32_t st) {
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const uint32_t w[4] = {kq[c].x, kq[c].y, kq[c].z, kq[c].w};
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        uint32_t a, b, d, e;
                        codes_to_halves<E4M3>(w[2 * half], a, b);
                        codes_to_halves<E4M3>(w[2 * half + 1], d, e);
                        const int key = blk * kKv8Block + 4 * (g >> 1) + (g & 1) + 2 * half;
                        sts16(smem + L::kK + st * L::kKStage + (c >> 1) * (kPageSize * 128) + key * 128 +
                                  (((((c & 1) << 2) + t4) ^ (key & 7)) << 4), a, b, d, e);
                    }
                }
                proxy_fence();
                __syncwarp();
                if (lane == 0) mb_arrive(&k_full[st]);
            };
            // V^T rows: dimension 32 c + 4 g + i, keys 16 blk + 4 t4 .. + 3; positions
            // behind the sequence may hold anything, an E4M3 NaN too
            float vref = 0.0f, vtop = 0.0f;
            auto write_v = [&](uint32_t st, int j, const float4& vs4) {
                const int kb = k0 + j * kPageSize + blk * kKv8Block;
                vref = next_vref(vref, vtop, vscale_max(vs4, k0 + j * kPageSize, ctx + nb));
                const float vs = blk < 2 ? (blk ? vs4.y : vs4.x) : (blk == 2 ? vs4.z : vs4.w);
                const float ratio = kb < ctx + nb ? vs * pow2_inv(vref) * kVUp : 0.0f;
                const int left = ctx + nb - kb - 4 * t4;
                const uint32_t keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
                const __half2 rr = __floats2half2_rn(ratio, ratio), ro = __floats2half2_rn(-1152.0f * ratio, -1152.0f * ratio);
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const uint32_t w[4] = {vq[c].x, vq[c].y, vq[c].z, vq[c].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t a, b;
                        scaled_halves<E4M3>(E4M3 ? w[i] & keep : w[i], rr, ro, a, b);
                        const int d = c * 32 + 4 * g + i;
                        sts8(smem + L::kV + st * L::kVStage + d * 128 + (((2 * blk + (t4 >> 1)) ^ (d & 7)) << 4) + (t4 & 1) * 8, a, b);
                    }
                }
                proxy_fence();
                __syncwarp();
                if (lane == 0) mb_arrive(&v_full[st]);
            };
            bool ok = true;
            if (n > 0) {
                load_k(bt[0]);
                load_v();
            }
            for (int j = 0; j < n; j++) {
                const uint32_t J = J0 + j, st = J & 1, par = ((J >> 1) - 1) & 1;
                const float4 vs4 = next.v;
                const int after = next.page;   // of page j + 1
                next.load(p, bt, h, j + 1, n);
                if (J > 1 && !warp_wait(&k_empty[st], par, tl.wait_clocks)) { ok = false; break; }
                write_k(st);
                if (j + 1 < n) load_k(after);
                if (J > 1 && !warp_wait(&v_empty[st], par, tl.wait_clocks)) { ok = false; break; }
                write_v(st, j, vs4);
                if (j + 1 < n) load_v();
            }
            if (!ok && lane == 0) atomicOr(&bad_s, 1);
        } else if (warp == 12 && lane == 0) {
            // ------------------------------------------------------ products
            int fail = fail_s;
            auto scores = [&](int tile, int j) -> bool {   // S of page j of a tile
                const uint32_t J = J0 + j, T = (tile ? jt1 : jt0) + j;
                // over P of the tile's page before last: its product has to be done (the
                // items before are; their phase could be mistaken for a later one's)
                if (j > 1 && !mb_wait(&bars[tile].pv_done, (T - 2) & 1, tl.wait_clocks)) return false;
                if (j == 0 && !mb_wait(&bars[tile].q_full, (tile ? items1 : items0) & 1, tl.wait_clocks)) return false;
                if (!mb_wait(&k_full[J & 1], (J >> 1) & 1, tl.wait_clocks)) return false;
                if (fail && --fail == 0) return false;
                tc_after();
#pragma unroll
                for (int q = L::kParts - 1; q >= 0; q--)   // the remainders first, while the sums are small
#pragma unroll
                    for (int k = 0; k < HD / 16; k++)
                        umma_f16<kPageSize>(tmem + tile * 256 + (T & 1) * 64,
                                            desc_sw128(smem + L::kQ + tile * L::kQTile + q * L::kQPart +
                                                       (k >> 2) * (kRows * 128) + (k & 3) * 32),
                                            desc_sw128(smem + L::kK + (J & 1) * L::kKStage +
                                                       (k >> 2) * (kPageSize * 128) + (k & 3) * 32),
                                            q < L::kParts - 1 || k > 0);
                umma_commit(&bars[tile].s_full[T & 1]);
                if (tile == nt - 1) umma_commit(&k_empty[J & 1]);
                return true;
            };
            auto output = [&](int tile, int j) -> bool {   // O (+)= P V of page j of a tile
                const uint32_t J = J0 + j, T = (tile ? jt1 : jt0) + j;
                if (!mb_wait(&v_full[J & 1], (J >> 1) & 1, tl.wait_clocks) ||
                    !mb_wait(&bars[tile].p_full[T & 1], (T >> 1) & 1, tl.wait_clocks))
                    return false;
                if (fail && --fail == 0) return false;
                tc_after();
#pragma unroll
                for (int q = L::kParts - 1; q >= 0; q--)
#pragma unroll
                    for (int k = 0; k < kPageSize / 16; k++)
                        umma_f16_ta<HD>(tmem + tile * 256 + 128, tmem + tile * 256 + (T & 1) * 64 + q * 16 + (k >> 1) * 32 + (k & 1) * 8,
                                        desc_sw128(smem + L::kV + (J & 1) * L::kVStage + k * 32), (F32 ? j % kFold : j) > 0 || q < L::kParts - 1 || k > 0);
                umma_commit(&bars[tile].pv_done);
                if (tile == nt - 1) umma_commit(&v_empty[J & 1]);
                return true;
            };
            bool ok = true;
            if (n > 0)
                ok = scores(0, 0) && (nt == 1 || scores(1, 0));
            for (int j = 0; j < n && ok; j++) {
                ok = (j + 1 >= n || scores(0, j + 1)) && output(0, j);
                if (nt > 1) ok = ok && (j + 1 >= n || scores(1, j + 1)) && output(1, j);
            }
            fail_s = fail;
            if (!ok) atomicOr(&bad_s, 1);
        }
        __syncthreads();
        if (bad_s) break;
        J0 += n;
        jt0 += n;
        items0 += n > 0;
        if (nt > 1) {
            jt1 += n;
            items1 += n > 0;
        }
        if (it.splits > 1) range_done(tl, it, joins);
        __syncthreads();
    }
    __syncthreads();
    if (bad_s) {
        // products under way read this CTA's memory and write its TMEM, whichever wait
        // ran out: all that were issued signal `drained`
        if (warp == 12 && lane == 0) {
            atomicOr(&g_kv8_error, 1);
            umma_commit(&drained);
            (void)mb_wait(&drained, 0, tl.wait_clocks);
        }
        // the tiles that other CTAs share with this one are not joined, by none of them,
        // and their counts start from zero again
        if (warp == 0)
            while (it.pages) {
                if (lane == 0 && it.splits > 1) (void)arrive_last(tl, it, kGivenUp);
                const long long x = it.next;
                __syncwarp();
                next_item(p, tl, x, lane, it);
                __syncwarp();
            }
        __syncthreads();
    }
    if (warp == 12) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
    // the tiles that this CTA completed, each from its ranges in their order
    __threadfence();
    for (int k = 0; k < joins.n && !bad_s; k++) {
        const Kv8Item& jt = joins.item[k];
        join_tile<HD, kThreads, kPair>(tl, jt, min(kPair, jt.nb * p.group - jt.tile * kPair), [&](int r, int d, const float (&acc)[4]) {
            const int pr = jt.tile * kPair + r, tk = pr / p.group;
            const int hq = jt.head * p.group + pr - tk * p.group;
            if (jt.row0 + tk < p.rows)
                store4<DT>(p.out, (size_t)(jt.row0 + tk) * p.ldo + (size_t)hq * HD + d, vec, acc);
        });
    }
}

template <class F>
cudaError_t with_kernel(int hd, int type, int dtype, F f) {
#define FL_KV8_K(HD)                                                                                            \
    if (hd == HD) {                                                                                             \
        if (type == FL_KV8_E4M3)                                                                                \
            return dtype == FL_F32   ? f(kv8_prefill_kernel<HD, FL_F32, true>, Layout<HD, true>::kBytes)        \
                   : dtype == FL_F16 ? f(kv8_prefill_kernel<HD, FL_F16, true>, Layout<HD, false>::kBytes)       \
                                     : f(kv8_prefill_kernel<HD, FL_BF16, true>, Layout<HD, false>::kBytes);     \
        return dtype == FL_F32   ? f(kv8_prefill_kernel<HD, FL_F32, false>, Layout<HD, true>::kBytes)           \
               : dtype == FL_F16 ? f(kv8_prefill_kernel<HD, FL_F16, false>, Layout<HD, false>::kBytes)          \
                                 : f(kv8_prefill_kernel<HD, FL_BF16, false>, Layout<HD, false>::kBytes);        \
    }
    FL_KV8_K(32)
    FL_KV8_K(64)
    FL_KV8_K(96)
    FL_KV8_K(128)
#undef FL_KV8_K
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t kv8_prefill_prepare(int head_dim, int type, int dtype) {
    return with_kernel(head_dim, type, dtype, [&](auto* k, int smem) {
        return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    });
}

cudaError_t launch_kv8_prefill(const Kv8AttnParams& p, const Kv8Tiles& tl, int ctas, cudaStream_t s) {
    const int es = p.dtype == FL_F32 ? 4 : 2;
    const int vec = ((uintptr_t)p.q & 15) == 0 && ((uintptr_t)p.out & 15) == 0 && p.ldq * es % 16 == 0 &&
                    p.ldo * es % 16 == 0;
    g_kv8_launched.store(true, std::memory_order_relaxed);
    return with_kernel(p.head_dim, p.type, p.dtype, [&](auto* k, int smem) {
        k<<<ctas, kThreads, smem, s>>>(p, tl, vec);
        return cudaGetLastError();
    });
}

int take_kv8_error() {
    int v = 0;
    if (!g_kv8_launched.load(std::memory_order_relaxed)) return 0;   // no wait could give up: no copy
    if (cudaMemcpyFromSymbol(&v, g_kv8_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) {
        const int z = 0;
        cudaMemcpyToSymbol(g_kv8_error, &z, sizeof(int));
    }
    return v;
}

}  // namespace fl
