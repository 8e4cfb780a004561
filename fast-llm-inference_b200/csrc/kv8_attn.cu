// Attention over the paged 8-bit KV cache (fl_kv8.h): query rows of a ragged
// batch against their sequences' pages, softmax online, sm_100a.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = e^(scale q_i . k_j - m_i)
//
// over the visible positions j, m_i a running reference of the maximum. Codes
// enter mma.m16n8k16 as halves (INT8 and E4M3 codes are exact there); a
// block's power-of-two scales multiply its scores, and its probabilities,
// exactly. Rows of 8 dimensions and of 4 positions lie in the cache in the
// products' operand order, so a warp reads a block of 16 positions with one
// 16-byte copy per lane and 32 dimensions, through its own slots in shared memory.
//
// Queries enter as halves too, each row shifted by a power of two so that its
// largest value lies in [2^14, 2^15): exact for fp16 and bf16 rows down to
// 2^-29 of the row's largest value. An f32 row enters as two halves (value and
// remainder, 22 bits together): a tile then holds 8 rows, their remainders in
// the tile's other 8 rows, so the second half costs no further product. The
// probabilities of f32 rows are split the same way. Those of 16-bit rows enter as one
// half, off by 2^-11 of themselves: no more than the output's own rounding (fp16;
// bf16 2^-8), and a second half would cost as many products again.
//
// A product drops the bits of its sums below 2^-24, towards zero, so that sums over n
// blocks of a sign fall short by about n 2^-25 (30 k keys: 1.6e-5). f32 rows therefore add
// each block's products, rounded, to sums of their own; 16-bit rows, whose outputs round
// coarser, sum up in the products.
//
// Bound by the cache's bytes: 24 rows over 300 to 32000 keys (40 / 10 heads of 128,
// 0.91 GB) take 172 to 185 us, 75 to 81 % of the copy peak; 64 x 7 f32 rows over 1000 to
// 1500 keys (32 heads of 96, 0.53 GB) 114 us, 71 %. Loads straight into registers
// took 315 and 142 us: a warp waited for each block. Each warp takes one block of
// every page, so that nothing is shared before the tile's end.
#include <math.h>

#include <algorithm>

#include "fl_common.cuh"
#include "fl_kv8.h"
#include "fl_kv8_attn.cuh"
#include "fl_kv8_types.cuh"

namespace fl {

namespace {

constexpr int kAW = 4;   // warps per CTA: one per 16-position block of a page
constexpr int kStages = 4;   // blocks in flight or in use per warp
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The products alone, of rows 0 - 7 and 8 - 15 together, added to d rounded.
__device__ __forceinline__ void mma16816_rounded(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    float x[4];
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    d[0] += x[0] + x[2];
    d[1] += x[1] + x[3];
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float2 lds8(uint32_t a) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

template <int HD, int DT, bool E4M3>
__global__ void __launch_bounds__(kAW * 32, 3) kv8_attention_kernel(const Kv8AttnParams p, const Kv8Tiles tl, const int vec) {
    constexpr bool F32 = DT == FL_F32;
    constexpr int TR = F32 ? 8 : 16;   // query rows per tile
    constexpr int NC = HD / 32;
    constexpr int RR = F32 ? 1 : 2;    // rows of a thread
    constexpr int kStage = 2 * NC * 512 + 16;   // bytes: K, V, the two scales
    extern __shared__ __align__(128) uint8_t smem[];   // rings of the warps, then their results
    float(*o_s)[TR][HD] = reinterpret_cast<float(*)[TR][HD]>(smem);
    __shared__ float m_s[kAW][TR], l_s[kAW][TR];
    __shared__ Kv8Joins joins;
    if (threadIdx.x == 0) joins.n = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kStages * kStage);
    const int g = lane >> 2, t4 = lane & 3;
    __shared__ Kv8Item it;   // re-read where it is used: registers go to the tile
    for (long long x = -1;;) {
        if (warp == 0) next_item(p, tl, x, lane, it);
        __syncthreads();
        if (it.pages == 0) break;
        x = it.next;
        const int h = it.head, ctx = it.ctx, row0 = it.row0, nb = it.nb;
        const int np = min(TR, nb * p.group - it.tile * TR);       // packed rows of the tile
        const int tok_last = (it.tile * TR + np - 1) / p.group;
        const int kend = p.mask ? ctx + nb : ctx + tok_last + 1;   // positions any row may see
        // this thread's rows: token, query head
        int row[RR], tok[RR], head[RR];
        bool live[RR];
#pragma unroll
        for (int r = 0; r < RR; r++) {
            const int pr = it.tile * TR + g + 8 * r;
            tok[r] = pr / p.group;
            head[r] = h * p.group + pr - tok[r] * p.group;
            row[r] = row0 + tok[r];
            live[r] = g + 8 * r < np && row[r] < p.rows;
        }
        // queries, shifted, as operand fragments: k step s of chunk c holds
        // dimensions 32 c + 8 t4 + 4 s .. + 3
        uint32_t qa[NC][2][4];
        float unshift[RR];
#pragma unroll
        for (int r = 0; r < RR; r++) {
            float amax = 0.0f;
            float f[NC][8];
#pragma unroll
            for (int c = 0; c < NC; c++) {
#pragma unroll
                for (int j = 0; j < 8; j++) f[c][j] = 0.0f;
                if (live[r]) load8<DT>(p.q, (size_t)row[r] * p.ldq + (size_t)head[r] * HD + c * 32 + t4 * 8, vec, f[c]);
#pragma unroll
                for (int j = 0; j < 8; j++) amax = fabsf(f[c][j]) > amax || f[c][j] != f[c][j] ? fabsf(f[c][j]) : amax;
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const float sh = row_shift(amax);
            unshift[r] = pow2_inv(sh) * p.scale;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) y[j] = f[c][4 * s + j] * sh;
                    qa[c][s][r] = h2(y[0], y[1]);
                    qa[c][s][2 + r] = h2(y[2], y[3]);
                    if constexpr (F32) {
#pragma unroll
                        for (int j = 0; j < 4; j++) y[j] -= __half2float(__float2half_rn(y[j]));
                        qa[c][s][1] = h2(y[0], y[1]);
                        qa[c][s][3] = h2(y[2], y[3]);
                    }
                }
        }
        float m[RR], l[RR];
        float o[NC][4][4];
        float vref = 0.0f, vtop = 0.0f;   // scale of the accumulators (next_vref)
#pragma unroll
        for (int r = 0; r < RR; r++) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[c][j][i] = 0.0f;

        // this warp's blocks: one a page, up to the last visible position. They
        // pass through a ring in shared memory; every lane copies the very 16
        // bytes that it will read, so a warp waits for its own copies alone
        const int* bt = p.t.block_table + (size_t)it.seq * p.max_pages + it.page0;
        const int nblk = min(it.pages, (kend - it.page0 * kPageSize - warp * kKv8Block + kPageSize - 1) / kPageSize);
        int pages = lane < nblk ? bt[lane] : 0;   // of 32 blocks at a time, one a lane
        auto fetch = [&](int i) {
            if (i < nblk) {
                if (i && (i & 31) == 0) pages = i + lane < nblk ? bt[i + lane] : 0;
                const size_t ph = (size_t)__shfl_sync(0xffffffffu, pages, i & 31) * p.kv_heads + h;
                const size_t off = ph * (kPageSize * HD) + warp * (kKv8Block * HD) + lane * 16;
                const uint32_t d = ring + (i % kStages) * kStage + lane * 16;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    cp_async16(d + c * 512, p.k + off + c * 512);
                    cp_async16(d + (NC + c) * 512, p.v + off + c * 512);
                }
                if (lane < 2) cp_async4(ring + (i % kStages) * kStage + 2 * NC * 512 + lane * 4,
                                        (lane ? p.vs : p.ks) + ph * kKv8Sub + warp);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) fetch(i);
        for (int i = 0; i < nblk; i++) {
            const int pos0 = (it.page0 + i) * kPageSize + warp * kKv8Block;
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();   // the scales come from lanes 0 and 1; slot i - 1 has been read
            const uint32_t st = ring + (i % kStages) * kStage;
            uint4 kq[NC], vq[NC];
#pragma unroll
            for (int c = 0; c < NC; c++) {
                kq[c] = lds16(st + c * 512 + lane * 16);
                vq[c] = lds16(st + (NC + c) * 512 + lane * 16);
            }
            const float2 sc = lds8(st + 2 * NC * 512);
            const float ks = sc.x, vs = sc.y;
            fetch(i + kStages - 1);
            // positions behind the sequence may hold anything: an E4M3 byte there may be a NaN
            if (E4M3 && pos0 + kKv8Block > ctx + nb) {
                const int lim = ctx + nb - pos0 - 4 * t4;   // of this lane's four V positions
                const uint32_t keep = lim >= 4 ? 0xffffffffu : lim <= 0 ? 0u : (1u << (8 * lim)) - 1u;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    vq[c].x &= keep; vq[c].y &= keep; vq[c].z &= keep; vq[c].w &= keep;
                }
            }
            float sa[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int c = 0; c < NC; c++) {
                uint32_t b0, b1;
                codes_to_halves<E4M3>(kq[c].x, b0, b1);
                mma16816(sa[0], qa[c][0], b0, b1);
                codes_to_halves<E4M3>(kq[c].z, b0, b1);
                mma16816(sa[1], qa[c][0], b0, b1);
                codes_to_halves<E4M3>(kq[c].y, b0, b1);
                mma16816(sa[0], qa[c][1], b0, b1);
                codes_to_halves<E4M3>(kq[c].w, b0, b1);
                mma16816(sa[1], qa[c][1], b0, b1);
            }
            // scores (base 2) of row r at positions pos0 + 4 t4 + 2 half + e
            float s[RR][4];
#pragma unroll
            for (int r = 0; r < RR; r++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float* a = sa[e >> 1];
                    const float raw = F32 ? a[e & 1] + a[2 + (e & 1)] : a[2 * r + (e & 1)];
                    s[r][e] = raw * ks * unshift[r];
                }
            if (p.mask || pos0 + kKv8Block > ctx) {
#pragma unroll
                for (int r = 0; r < RR; r++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = pos0 + 4 * t4 + e - ctx;   // new row, negative: cached
                        bool see = j <= tok[r];
                        if (p.mask && j >= 0) see = j < min(nb, p.ldm) && live[r] && p.mask[(size_t)row[r] * p.ldm + j] != 0;
                        if (!see) s[r][e] = -INFINITY;
                    }
            }
            // reference of the maximum, and of the V scale
            float mx[RR];
            bool move = vref_moves(vref, vs);
#pragma unroll
            for (int r = 0; r < RR; r++) {
                mx[r] = fmaxf(fmaxf(s[r][0], s[r][1]), fmaxf(s[r][2], s[r][3]));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                move |= mx[r] > m[r] + kSlack || (m[r] == -INFINITY && mx[r] > m[r]);
            }
            if (__any_sync(0xffffffffu, move)) {
                const float vnew = next_vref(vref, vtop, vs);
                const float vr = vref * pow2_inv(vnew);
                vref = vnew;
#pragma unroll
                for (int r = 0; r < RR; r++) {
                    const float mn = fmaxf(m[r], mx[r]);
                    const float al = m[r] == -INFINITY ? 0.0f : ex2(m[r] - mn);
                    m[r] = mn;
                    l[r] *= al;
                    const float f = al * vr;
#pragma unroll
                    for (int c = 0; c < NC; c++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            o[c][j][2 * r] *= f;
                            o[c][j][2 * r + 1] *= f;
                        }
                }
            }
            uint32_t pa[4];
            const float vf = vs * pow2_inv(vref);
#pragma unroll
            for (int r = 0; r < RR; r++) {
                const float mr = m[r] == -INFINITY ? 0.0f : m[r] - kShift;
                float pr[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    pr[e] = ex2(s[r][e] - mr);
                    l[r] += pr[e];
                    pr[e] *= vf;
                }
                pa[r] = h2(pr[0], pr[1]);
                pa[2 + r] = h2(pr[2], pr[3]);
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 4; e++) pr[e] -= __half2float(__float2half_rn(pr[e]));
                    pa[1] = h2(pr[0], pr[1]);
                    pa[3] = h2(pr[2], pr[3]);
                }
            }
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const uint32_t vw[4] = {vq[c].x, vq[c].y, vq[c].z, vq[c].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t b0, b1;
                    codes_to_halves<E4M3>(vw[j], b0, b1);
                    if constexpr (F32) mma16816_rounded(o[c][j], pa, b0, b1);
                    else mma16816(o[c][j], pa, b0, b1);
                }
            }
        }
        // this warp's result: reference, sum, normalised output
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RR; r++) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const float f = l[r] != 0.0f ? __fdiv_rn(vref, l[r]) : 0.0f;   // NaN sums stay NaN
            if (t4 == 0) {
                m_s[warp][g + 8 * r] = m[r];
                l_s[warp][g + 8 * r] = l[r];
            }
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float4 v;
                    float* vp = reinterpret_cast<float*>(&v);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        vp[j] = o[c][j][2 * r + e] * f;
                    *reinterpret_cast<float4*>(&o_s[warp][g + 8 * r][c * 32 + 8 * t4 + 4 * e]) = v;
                }
        }
        __syncthreads();
        // joined over the warps: the weights are l 2^(m - M)
        // slots of a part: its first range, of a tile begun before it, and its last
        const size_t slot = 2 * (size_t)blockIdx.x + (it.split == 0);
        for (int idx = threadIdx.x; idx < np * (HD / 4); idx += kAW * 32) {
            const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int k = 0; k < kAW; k++) M = fmaxf(M, m_s[k][r]);
            float L = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kAW; k++) {
                if (l_s[k][r] == 0.0f) continue;
                const float wk = l_s[k][r] * ex2(m_s[k][r] - M);
                L += wk;
                const float4 v = *reinterpret_cast<const float4*>(&o_s[k][r][d]);
                acc[0] += wk * v.x; acc[1] += wk * v.y; acc[2] += wk * v.z; acc[3] += wk * v.w;
            }
            const float f = L != 0.0f ? __fdiv_rn(1.0f, L) : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] *= f;
            if (it.splits > 1) {
                *reinterpret_cast<float4*>(tl.part + (slot * TR + r) * HD + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                if (d == 0) tl.part_ml[slot * TR + r] = make_float2(M, L);
            } else {
                const int pr = it.tile * TR + r, tk = pr / p.group;
                const int hq = h * p.group + pr - tk * p.group;
                if (row0 + tk < p.rows) store4<DT>(p.out, (size_t)(row0 + tk) * p.ldo + (size_t)hq * HD + d, vec, acc);
            }
        }
        if (it.splits > 1) range_done(tl, it, joins);
        __syncthreads();
    }
    // the tiles that this CTA completed, each from its ranges in their order
    __threadfence();
    for (int k = 0; k < joins.n; k++) {
        const Kv8Item& jt = joins.item[k];
        join_tile<HD, kAW * 32, TR>(tl, jt, min(TR, jt.nb * p.group - jt.tile * TR), [&](int r, int d, const float (&acc)[4]) {
            const int pr = jt.tile * TR + r, tk = pr / p.group;
            const int hq = jt.head * p.group + pr - tk * p.group;
            if (jt.row0 + tk < p.rows)
                store4<DT>(p.out, (size_t)(jt.row0 + tk) * p.ldo + (size_t)hq * HD + d, vec, acc);
        });
    }
}

// Calls f with the kernel of a configuration.
template <class F>
cudaError_t with_kernel(int hd, int type, int dtype, F f) {
#define FL_KV8_K(HD)                                                                                           \
    if (hd == HD) {                                                                                            \
        if (type == FL_KV8_E4M3)                                                                               \
            return dtype == FL_F32   ? f(kv8_attention_kernel<HD, FL_F32, true>)                               \
                   : dtype == FL_F16 ? f(kv8_attention_kernel<HD, FL_F16, true>)                               \
                                     : f(kv8_attention_kernel<HD, FL_BF16, true>);                             \
        return dtype == FL_F32   ? f(kv8_attention_kernel<HD, FL_F32, false>)                                  \
               : dtype == FL_F16 ? f(kv8_attention_kernel<HD, FL_F16, false>)                                  \
                                 : f(kv8_attention_kernel<HD, FL_BF16, false>);                                \
    }
    FL_KV8_K(32)
    FL_KV8_K(64)
    FL_KV8_K(96)
    FL_KV8_K(128)
#undef FL_KV8_K
    return cudaErrorInvalidValue;
}

}  // namespace

// Dynamic shared memory: the rings, later the warps' results.
int attention_smem(int hd, int dtype) {
    const int ring = kAW * kStages * (2 * (hd / 32) * 512 + 16);
    return std::max(ring, kAW * (dtype == FL_F32 ? 8 : 16) * hd * 4);
}

int kv8_attention_occupancy(int head_dim, int type, int dtype) {
    int n = 0;
    const int smem = attention_smem(head_dim, dtype);
    with_kernel(head_dim, type, dtype, [&](auto* k) {
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, kAW * 32, smem);
        return e;
    });
    return n > 0 ? n : 1;
}

cudaError_t launch_kv8_attention(const Kv8AttnParams& p, const Kv8Tiles& tl, int ctas, cudaStream_t s) {
    const int es = p.dtype == FL_F32 ? 4 : 2;
    const int vec = ((uintptr_t)p.q & 15) == 0 && ((uintptr_t)p.out & 15) == 0 && p.ldq * es % 16 == 0 &&
                    p.ldo * es % 16 == 0;
    return with_kernel(p.head_dim, p.type, p.dtype, [&](auto* k) {
        k<<<ctas, kAW * 32, attention_smem(p.head_dim, p.dtype), s>>>(p, tl, vec);
        return cudaGetLastError();
    });
}

}  // namespace fl
