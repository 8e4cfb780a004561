// Shared by the attention kernels over the 8-bit KV cache (kv8_attn.cu,
// kv8_prefill.cu): conversions, the distribution of the work and the join of a
// tile's ranges.
#pragma once

#include <math.h>

#include "fl_common.cuh"
#include "fl_kv8.h"
#include "fl_kv8_types.cuh"

namespace fl {

constexpr float kTileCost = 3.0f, kJoinCost = 20.0f;   // in pages, see next_item
constexpr float kShift = 7.0f;   // probabilities enter as 2^7 p: 2^-21 of the largest is a normal half
constexpr float kSlack = 8.0f;   // the reference follows the maximum once it lags by 2^8

// The accumulators' scale is that of a V block (row kernel) or page (prefill kernel) met
// so far. It follows a larger one, and one that lies more than 2^8 below it: what enters
// as halves carries the ratio of the two, and bits below 2^-24 are lost. It stays within
// 2^60 of the largest, vtop, where the sums are finite, and at a scale, 2^-100 or more.
constexpr float kVSlack = 0x1p-8f;
__device__ __forceinline__ bool vref_moves(float vref, float vs) { return vs > vref || vs < vref * kVSlack; }
__device__ __forceinline__ float next_vref(float vref, float& vtop, float vs) {
    vtop = fmaxf(vtop, vs);
    return vref_moves(vref, vs) ? fmaxf(vs, fmaxf(vtop * 0x1p-60f, 0x1p-100f)) : vref;
}

// 2^x, about 2 units in the last place; 0 far below.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Four codes of a word as two half pairs.
template <bool E4M3>
__device__ __forceinline__ void codes_to_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (E4M3) {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
        const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// 8 values at dimensions d .. d + 7 of a query row.
template <int DT>
__device__ __forceinline__ void load8(const void* q, size_t i, int vec, float (&f)[8]) {
    float a[4], b[4];
    load4<DT>(q, i, vec, a);
    load4<DT>(q, i + 4, vec, b);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        f[j] = a[j];
        f[4 + j] = b[j];
    }
}

// A range of a tile's pages.
struct Kv8Item {
    int seq, head, ctx, row0, nb;
    int tile, page0, pages;   // no pages: none is left
    int split, splits;        // this range among the tile's
    int part;                 // the part that holds the tile's first page
    long long next;           // where the CTA goes on
};

// The sequence whose work x falls into: start[b] <= x < start[b + 1]. A warp
// narrows the range 32-fold a step.
__device__ __forceinline__ int find_work(const long long* start, int nseq, long long x, int lane) {
    int lo = 0, n = nseq;   // start[lo] <= x < start[lo + n]
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int at = lo + lane * step;
        const bool below = lane * step < n && start[at] <= x;
        const int k = 31 - __clz((int)__ballot_sync(0xffffffffu, below));
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// The work of a CTA, item by item (x: where it stands, -1 at first); by a warp.
// Two ways to share it. Whole tiles, CTA by CTA; or the (kv head, row tile,
// page) triples, in that order, cut into equal parts, one a CTA, which end
// together whatever the lengths are, while a tile that several parts share is
// joined by the last of them to arrive. What each takes is estimated in pages:
// kTileCost a tile, kJoinCost for the joins. At 64 x 32 tiles of 21 pages whole
// tiles took 106 us and parts 120; at 24 x 10 tiles of 5 to 500, 290 and 168; in the
// prefill kernel at 10 tiles of 11 pages, 45 and 74.
__device__ __forceinline__ void next_item(const Kv8AttnParams& p, const Kv8Tiles& tl, long long x, int lane,
                                          Kv8Item& out) {
    const Kv8Meta& mt = *p.t.meta;
    const long long tiles = mt.list[tl.list].tiles, work = mt.list[tl.list].work, G = gridDim.x;
    const float mean = (float)work / (float)max(1ll, tiles), per_cta = (float)(tiles * p.kv_heads) / (float)G;
    const bool whole = ceilf(per_cta) * (mean + kTileCost) + ((float)mt.list[tl.list].max_pages - mean) <=
                       per_cta * mean + (per_cta + 1.0f) * kTileCost + kJoinCost;
    const long long total = (whole ? tiles : work) * p.kv_heads;
    // a prefill part of n pages takes about 2 n us, and its share of a join 1.3
    const int least = tl.list ? (int)ceilf(sqrtf(0.65f * mean)) : 1;
    const long long size = whole ? 1 : max((long long)least, (total + G - 1) / G);
    if (x < 0) x = (long long)blockIdx.x * size;
    Kv8Item it = {};
    if (x < (whole ? total : min(total, (blockIdx.x + 1ll) * size))) {
        it.head = (int)(x / (whole ? tiles : work));
        const long long in_head = x - it.head * (whole ? tiles : work);
        const long long* start = whole ? tl.tile_start : tl.work_start;
        it.seq = find_work(start, mt.seqs, in_head, lane);
        const long long in_seq = in_head - start[it.seq];
        it.ctx = p.t.ctx[it.seq];
        it.row0 = p.t.row_start[it.seq];
        it.nb = p.t.row_start[it.seq + 1] - it.row0;
        it.pages = (it.ctx + it.nb + kPageSize - 1) / kPageSize;
        it.splits = 1;
        if (whole) {
            it.tile = (int)in_seq;
            it.next = x + G;
        } else {
            const int tile_pages = it.pages;
            it.tile = (int)(in_seq / tile_pages);
            it.page0 = (int)(in_seq - (long long)it.tile * tile_pages);
            it.pages = (int)min((long long)(tile_pages - it.page0), (blockIdx.x + 1ll) * size - x);
            const long long tile_x = x - it.page0;   // the tile's first triple
            it.part = (int)(tile_x / size);
            it.splits = (int)((tile_x + tile_pages - 1) / size) - it.part + 1;
            it.split = (int)blockIdx.x - it.part;
            it.next = x + it.pages;
        }
    }
    if (lane == 0) out = it;
}

// Shift of a row with largest magnitude a: a 2^sh in [2^14, 2^15); 0 for a
// zero row and for one that is not finite (its results are NaN).
__device__ __forceinline__ float row_shift(float a) {
    const int x = (int)((__float_as_uint(a) >> 23) & 255u);
    if (x == 0 || x == 255) return 1.0f;
    return __uint_as_float((uint32_t)min(max(127 + 14 - (x - 127), 1), 253) << 23);
}

// Tiles whose last range arrived in this CTA: of a part's two ranges that share
// a tile. They are joined at the kernel's end, where the loop's registers are free.
struct Kv8Joins {
    int n;
    Kv8Item item[2];
};
// A range arrives at its tile's count: the ranges so far, and above them those that
// were given up. The last one clears the count, for the launches that follow; true
// for it if all ranges have their results.
constexpr int kGivenUp = 1 << 16;   // above any number of ranges
__device__ __forceinline__ bool arrive_last(const Kv8Tiles& tl, const Kv8Item& it, int given_up) {
    const int n = atomicAdd(tl.part_cnt + it.part, 1 + given_up) + given_up;
    if ((n & (kGivenUp - 1)) != it.splits - 1) return false;
    tl.part_cnt[it.part] = 0;
    return n < kGivenUp;
}
// After a range's results are written (whole block).
__device__ __forceinline__ void range_done(const Kv8Tiles& tl, const Kv8Item& it, Kv8Joins& joins) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0 && arrive_last(tl, it, 0)) joins.item[joins.n++] = it;
}

// Rows 0 .. np - 1 of a tile joined from its parts' results, in the parts' order,
// by a block of NT threads; put(row, dimension, four values). First some lanes
// a row turn (m, l) into the parts' weights l 2^(m - M) and the row's 1 / sum, in
// place (the last to arrive is alone with them); then the loads of the results do not
// wait on each other. Weights within the loop over the results, one load
// behind the other, made the join the longest part of a call over few tiles: 256
// rows x 10 heads over 16 k keys took 301 us, now 128.
template <int HD, int NT, int ROWS, class Put>
__device__ __forceinline__ void join_tile(const Kv8Tiles& tl, const Kv8Item& it, int np, Put put) {
    constexpr int U = 8;   // results under way
    constexpr int GL = NT / ROWS >= 16 ? 16 : NT / ROWS >= 8 ? 8 : 1;   // lanes of a row
    static_assert(NT >= GL * ROWS, "a row for every group of lanes");
    // slots of a part: its first range, of a tile begun before it, and its last
    auto at = [&](int k, int r) { return (2 * (size_t)(it.part + k) + (k == 0)) * ROWS + r; };
    const int row = threadIdx.x / GL, first = row < np ? (int)threadIdx.x % GL : it.splits;
    float M = -INFINITY, L = 0.0f;
#pragma unroll 4
    for (int k = first; k < it.splits; k += GL) M = fmaxf(M, __ldcg(&tl.part_ml[at(k, row)]).x);
#pragma unroll
    for (int o = GL / 2; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    for (int k0 = first; k0 < it.splits; k0 += 4 * GL) {
        float2 ml[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
            ml[u] = k0 + u * GL < it.splits ? __ldcg(&tl.part_ml[at(k0 + u * GL, row)]) : make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const float w = ml[u].y != 0.0f ? ml[u].y * ex2(ml[u].x - M) : 0.0f;   // NaN sums stay NaN
            L += w;
            if (k0 + u * GL < it.splits) tl.part_ml[at(k0 + u * GL, row)].x = w;
        }
    }
#pragma unroll
    for (int o = GL / 2; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (first == 0 && row < np) tl.part_ml[at(0, row)].y = L != 0.0f ? __fdiv_rn(1.0f, L) : 0.0f;
    __syncthreads();
    for (int idx = threadIdx.x; idx < np * (HD / 4); idx += NT) {
        const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
        float acc[4] = {0.f, 0.f, 0.f, 0.f}, f = 0.0f;
        for (int k0 = 0; k0 < it.splits; k0 += U) {
            float2 wf[U];
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                wf[u] = make_float2(0.f, 0.f);
                if (k0 + u < it.splits) {
                    wf[u] = __ldcg(&tl.part_ml[at(k0 + u, r)]);
                    v[u] = __ldcg(reinterpret_cast<const float4*>(tl.part + at(k0 + u, r) * HD + d));
                }
            }
            if (k0 == 0) f = wf[0].y;
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (wf[u].x == 0.0f) continue;
                acc[0] += wf[u].x * v[u].x; acc[1] += wf[u].x * v[u].y;
                acc[2] += wf[u].x * v[u].z; acc[3] += wf[u].x * v[u].w;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) acc[j] *= f;
        put(r, d, acc);
    }
}

}  // namespace fl
