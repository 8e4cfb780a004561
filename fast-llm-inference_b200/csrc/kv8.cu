// Paged KV cache in 8 bits for ragged batches: the handle, the plan (block
// tables, slot maps and work lists from request lengths), the append and the
// gather. The rules are stated in include/fl_cuda.h.
#include <string.h>

#include <algorithm>
#include <new>

#include "fl_common.cuh"
#include "fl_kv8.h"
#include "fl_kv8_types.cuh"
#include "fl_runtime.h"

namespace fl {

namespace {

// ---------------------------------------------------------------------------
// Plan: one kernel, of one CTA, or of one cluster of eight where a prompt batch
// has rows for them. CTA 0 checks the lengths and scans them (each thread holds
// one sequence while there are no more of them than threads); then all threads
// return and take pages and write the row maps, item by item: an item's sequence
// is found by bisection in the starts, which lie in shared memory up to
// 1024 sequences. Bound by latency: the loads of the lengths, two barriers of the scan, the
// page loads and stores with a barrier after each: 4.9 us for 8 sequences of one row;
// 20 us each to drop and to admit 1021 sequences with 33 k pages and 40 k rows.
// ---------------------------------------------------------------------------
constexpr int kSmSeqs = 1024;   // sequences whose starts shared memory holds

// Packed query rows of a sequence (new rows x heads per kv head) from which the
// prefill kernel takes it. 128 / 188 rows in 16 bits: 4 sequences x 3700 keys (10 kv
// heads x 128) 71 / 90 us, the row kernel 77 / 103; 1 x 16 k 82 / 107, 77 / 101; 32 x 1000
// 127 / 157, 169 / 251; one of 600 keys 33 / 43, 17 / 19. f32 (32 heads x 96) at 96 rows: 163,
// 175, 423 and 43 us, the row kernel 195, 193, 502 and 16; at 64 rows 159, 172, 401 and 43 to
// 135, 135, 325 and 16.
#ifndef FL_KV8_LONG_MIN
#define FL_KV8_LONG_MIN 192
#endif
#ifndef FL_KV8_LONG_MIN_F32
#define FL_KV8_LONG_MIN_F32 96
#endif
int long_min(const fl_kv8_t* h) { return h->c.dtype == FL_F32 ? FL_KV8_LONG_MIN_F32 : FL_KV8_LONG_MIN; }

struct PlanArgs {
    const int *ctx, *nw;
    Kv8Tables t;
    int nseq, max_new, max_pages, max_rows;
    int group, tile_rows, long_min;   // packed rows from which a sequence is on the second list
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct SeqPlan {
    int n, ctx, keep, need;   // new rows, cached positions, pages kept, pages held afterwards
    int rel;                  // pages returned
    bool bad;
};

__device__ __forceinline__ SeqPlan seq_plan(const PlanArgs& a, int b) {
    SeqPlan s;
    const int nw = a.nw[b], held = __ldcg(a.t.held + b), c = a.ctx[b];
    s.bad = false;
    s.n = max(nw, 0);
    s.ctx = 0;
    s.rel = nw < 0 ? held : 0;
    s.keep = nw < 0 ? 0 : held;
    s.need = s.keep;
    if (s.n > 0) {
        const long long n = (long long)c + s.n;
        s.bad = c < 0 || s.n > a.max_new || n > (long long)a.max_pages * kPageSize;
        if (!s.bad) {
            s.ctx = c;
            s.need = max(s.keep, (int)((n + kPageSize - 1) / kPageSize));
        }
    }
    return s;
}

// The first index b with start[b + 1] > r, start ascending, start[nseq] > r.
template <class At>
__device__ __forceinline__ int find_seq_by(int nseq, int r, At start) {
    int lo = 0, hi = nseq - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (start(mid + 1) > r) hi = mid; else lo = mid + 1;
    }
    return lo;
}
// What is summed over the sequences, in the order of the scan.
enum { V_ROWS, V_KEYS, V_REL, V_TAKE, V_UNITS, V_GBLK, V_TILES0, V_WORK0, V_TILES1, V_WORK1, V_COUNT };

__device__ __forceinline__ void add_seq(const PlanArgs& a, const SeqPlan& s, long long (&v)[V_COUNT], int (&mp)[2]) {
    const int n = s.n ? s.ctx + s.n : 0;
    v[V_ROWS] += s.n;
    v[V_KEYS] += n;
    v[V_REL] += s.rel;
    v[V_TAKE] += s.need - s.keep;
    v[V_UNITS] += s.n ? (n - 1) / kKv8Block - s.ctx / kKv8Block + 1 : 0;
    v[V_GBLK] += (n + kKv8Block - 1) / kKv8Block;
    const int li = s.n * a.group >= a.long_min, tr = li ? kKv8Long : a.tile_rows;
    const int tl = (s.n * a.group + tr - 1) / tr, pages = (n + kPageSize - 1) / kPageSize;
    v[li ? V_TILES1 : V_TILES0] += tl;
    v[li ? V_WORK1 : V_WORK0] += (long long)tl * pages;
    mp[li] = max(mp[li], pages);
}

// starts of sequence b's shares
__device__ __forceinline__ void put_starts(const Kv8Tables& t, int b, const long long (&v)[V_COUNT]) {
    t.row_start[b] = (int)v[V_ROWS];
    t.kv_start[b] = (int)v[V_KEYS];
    t.rel_start[b] = (int)v[V_REL];
    t.take_start[b] = (int)v[V_TAKE];
    t.unit_start[b] = (int)v[V_UNITS];
    t.gblk_start[b] = (int)v[V_GBLK];
    t.tile_start[0][b] = v[V_TILES0];
    t.work_start[0][b] = v[V_WORK0];
    t.tile_start[1][b] = v[V_TILES1];
    t.work_start[1][b] = v[V_WORK1];
}

template <int NT>
__global__ void __launch_bounds__(NT) kv8_plan_kernel(const PlanArgs a) {
    constexpr int NW = NT / 32;
    __shared__ long long part[V_COUNT][NW], total_s[V_COUNT];
    __shared__ int part_mp[2][NW], bad_s[NW];
    // row, release, take and unit starts, cached positions, pages kept
    __shared__ int sm[6][kSmSeqs + 1];
    uint32_t rank, nrank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nrank));
    const Kv8Tables& t = a.t;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool local = a.nseq <= kSmSeqs;
    if (rank == 0) {
        const int C = (a.nseq + NT - 1) / NT;
        const int b0 = min(a.nseq, (int)threadIdx.x * C), b1 = min(a.nseq, b0 + C);
        const int nfree = __ldcg(t.n_free);
        SeqPlan one = {};
        if (C == 1 && b0 < b1) one = seq_plan(a, b0);
        auto plan = [&](int b) { return C == 1 ? one : seq_plan(a, b); };
        long long own[V_COUNT] = {}, v[V_COUNT], tot[V_COUNT];
        int mp[2] = {}, bad = 0;
        for (int b = b0; b < b1; b++) {
            const SeqPlan s = plan(b);
            bad |= s.bad;
            add_seq(a, s, own, mp);
        }
        // exclusive prefixes over the threads: within the warp, then over the warps
#pragma unroll
        for (int i = 0; i < V_COUNT; i++) {
            long long inc = own[i];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            v[i] = inc - own[i];
            if (lane == 31) part[i][warp] = inc;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int m = __reduce_max_sync(0xffffffffu, mp[i]);
            if (lane == 0) part_mp[i][warp] = m;
        }
        bad = __any_sync(0xffffffffu, bad);
        if (lane == 0) bad_s[warp] = bad;
        __syncthreads();
        for (int i = warp; i < V_COUNT; i += NW) {   // each sum's warps by one of them
            const long long own_w = lane < NW ? part[i][lane] : 0;
            long long inc = own_w;
#pragma unroll
            for (int o = 1; o < NW; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            if (lane < NW) part[i][lane] = inc - own_w;
            if (lane == NW - 1) total_s[i] = inc;
        }
        bad = __any_sync(0xffffffffu, lane < NW && bad_s[lane]);
#pragma unroll
        for (int i = 0; i < 2; i++) mp[i] = __reduce_max_sync(0xffffffffu, lane < NW ? part_mp[i][lane] : 0);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V_COUNT; i++) {
            v[i] += part[i][warp];
            tot[i] = total_s[i];
        }
        const long long have = nfree + tot[V_REL];
        const int st = bad || tot[V_ROWS] > a.max_rows ? -1
                       : tot[V_TAKE] > have            ? (int)min(tot[V_TAKE] - have, 0x7fffffffll)
                                                       : 0;
        if (threadIdx.x == 0) {
            *t.status = st;
            *t.meta = st ? Kv8Meta{a.nseq, 0, 0, 0, 1, 0, {}}
                         : Kv8Meta{a.nseq, (int)tot[V_ROWS], (int)tot[V_UNITS], (int)tot[V_GBLK], 0, 0,
                                   {{tot[V_TILES0], tot[V_WORK0], mp[0]}, {tot[V_TILES1], tot[V_WORK1], mp[1]}}};
        }
        if (st != 0) {
            for (int b = threadIdx.x; b <= a.nseq; b += NT) t.row_start[b] = t.kv_start[b] = 0;
        } else {
            for (int b = b0; b < b1; b++) {
                const SeqPlan s = plan(b);
                put_starts(t, b, v);
                t.ctx[b] = s.ctx;
                if (local) {
                    sm[0][b] = (int)v[V_ROWS];
                    sm[1][b] = (int)v[V_REL];
                    sm[2][b] = (int)v[V_TAKE];
                    sm[3][b] = (int)v[V_UNITS];
                    sm[4][b] = s.ctx;
                    sm[5][b] = s.keep;
                }
                add_seq(a, s, v, mp);
            }
            if (threadIdx.x == 0) {
                put_starts(t, a.nseq, tot);
                if (local) {
                    sm[0][a.nseq] = (int)tot[V_ROWS];
                    sm[1][a.nseq] = (int)tot[V_REL];
                    sm[2][a.nseq] = (int)tot[V_TAKE];
                    sm[3][a.nseq] = (int)tot[V_UNITS];
                }
            }
        }
    }
    auto sync = [&]() {
        if (nrank > 1) cluster_sync(); else __syncthreads();
    };
    sync();
    if (__ldcg(&t.meta->refused)) return;   // nothing changes (every CTA alike)
    if (local && rank > 0) {   // the other CTAs' copies
        for (int b = threadIdx.x; b <= a.nseq; b += NT) {
            sm[0][b] = __ldcg(t.row_start + b);
            sm[1][b] = __ldcg(t.rel_start + b);
            sm[2][b] = __ldcg(t.take_start + b);
            sm[3][b] = __ldcg(t.unit_start + b);
            if (b < a.nseq) {
                sm[4][b] = __ldcg(t.ctx + b);
                sm[5][b] = a.nw[b] < 0 ? 0 : __ldcg(t.held + b);
            }
        }
        __syncthreads();
    }
    auto get = [&](int which, const int* g, int b) { return local ? sm[which][b] : __ldcg(g + b); };
    auto keep_of = [&](int b) { return local ? sm[5][b] : a.nw[b] < 0 ? 0 : __ldcg(t.held + b); };
    auto rows_at = [&](int b) { return get(0, t.row_start, b); };
    auto rel_at = [&](int b) { return get(1, t.rel_start, b); };
    auto take_at = [&](int b) { return get(2, t.take_start, b); };
    auto unit_at = [&](int b) { return get(3, t.unit_start, b); };
    const int i0 = (int)rank * NT + threadIdx.x, step = (int)nrank * NT;
    const int nrel = rel_at(a.nseq), ntake = take_at(a.nseq), top = __ldcg(t.n_free) + nrel;
    // returned pages: the first page of the first sequence ends on top
    if (nrel) {
        for (int i = i0; i < nrel; i += step) {
            const int b = find_seq_by(a.nseq, i, rel_at);
            t.free_pages[top - 1 - i] = __ldcg(t.block_table + (size_t)b * a.max_pages + i - rel_at(b));
        }
        sync();
    }
    for (int i = i0; i < ntake; i += step) {
        const int b = find_seq_by(a.nseq, i, take_at);
        t.block_table[(size_t)b * a.max_pages + keep_of(b) + i - take_at(b)] = __ldcg(t.free_pages + top - 1 - i);
    }
    const int nunit = unit_at(a.nseq);
    for (int i = i0; i < nunit; i += step) {
        const int b = find_seq_by(a.nseq, i, unit_at), u = i - unit_at(b);
        t.unit_row[i] = rows_at(b) + (u ? u * kKv8Block - get(4, t.ctx, b) % kKv8Block : 0);
    }
    sync();
    for (int b = i0; b < a.nseq; b += step) {   // a sequence without new rows has neither cached nor new pages to take
        const int k = keep_of(b) + take_at(b + 1) - take_at(b);
        t.held[b] = k;
    }
    if (i0 == 0) *t.n_free = top - ntake;
    const int rows = rows_at(a.nseq);
    for (int r = i0; r < rows; r += step) {
        const int b = find_seq_by(a.nseq, r, rows_at);
        const int p = get(4, t.ctx, b) + r - rows_at(b);
        t.pos[r] = p;
        t.row_seq[r] = b;
        t.slot[r] = __ldcg(t.block_table + (size_t)b * a.max_pages + p / kPageSize) * kPageSize + p % kPageSize;
    }
}

// Fresh tables: every page free (page 0 on top), nothing held.
__global__ void kv8_reset_kernel(const Kv8Tables t, int pages, int max_seqs) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < pages; i += gridDim.x * blockDim.x)
        t.free_pages[i] = pages - 1 - i;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < max_seqs; i += gridDim.x * blockDim.x) t.held[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *t.n_free = pages;
        *t.status = 0;
        *t.meta = Kv8Meta{};
    }
}

// ---------------------------------------------------------------------------
// Append: one warp per (16-position block touched, kv head, K or V). A lane
// holds the 16 codes of its 16 stored bytes per chunk of 32 dimensions (see
// fl_kv8.h), so the block's largest value is one warp reduction, and a stored
// piece is read, recoded where the scale grew, filled in and written whole.
// Bound by bytes: the rows once in, the codes once out; with the gather behind it
// 14 k bf16 rows of 10 x 128 take 77 us, the bytes of both 40.
// ---------------------------------------------------------------------------
struct AppendArgs {
    Kv8Tables t;
    const void *k, *v;
    size_t ldk, ldv;
    uint8_t *kc, *vc;
    float *ks, *vs;
    int rows, kv_heads, vec;
};

constexpr int kAppendWarps = 8;

// The lane's 16 values (or codes) of a chunk are four groups of four: group i
// of a K piece is position i / 2's dimensions 4 (i & 1) .. + 3 (the bytes of
// word i), of a V piece position i's four dimensions (byte i of every word).
template <bool V>
__device__ __forceinline__ int piece_pos(int lane, int i) {
    const int n = lane >> 2, t = lane & 3;
    return V ? 4 * t + i : 4 * (n >> 1) + (n & 1) + (i >> 1) * 2;
}
template <bool V>
__device__ __forceinline__ int piece_dim(int lane, int i) {
    return V ? (lane >> 2) * 4 : (lane & 3) * 8 + (i & 1) * 4;
}
// The bytes of word k that hold positions [first, first + m) of a block.
template <bool V>
__device__ __forceinline__ uint32_t piece_mask(int lane, int k, int first, int m) {
    if (!V) {
        const int p = piece_pos<false>(lane, k) - first;
        return p >= 0 && p < m ? 0xffffffffu : 0u;
    }
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int p = piece_pos<true>(lane, i) - first;
        b |= p >= 0 && p < m ? 0xffu << (8 * i) : 0u;
    }
    return b;
}

// Rows x[0 .. m) (row stride ld) into positions first .. first + m of a block.
template <int HD, int DT, bool E4M3, bool V>
__device__ __forceinline__ void append_block(const void* x, size_t at, size_t ld, int vec, int first, int m,
                                             uint8_t* code, float* sp, int lane) {
    constexpr int NC = HD / 32;
    float val[NC][16];
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p = piece_pos<V>(lane, i) - first;
            float f[4] = {0.f, 0.f, 0.f, 0.f};
            if (p >= 0 && p < m) load4<DT>(x, at + (size_t)p * ld + c * 32 + piece_dim<V>(lane, i), vec, f);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                val[c][4 * i + j] = f[j];
                const float y = fabsf(f[j]);
                amax = fmaxf(amax, y < INFINITY ? y : 0.0f);   // NaN and infinities set no scale
            }
        }
    float s = pow2_scale<E4M3>(warp_max(amax));
    const float s_old = first > 0 ? *sp : s;
    s = fmaxf(s, s_old);
    const bool grew = s > s_old;
    const float inv = pow2_inv(s), ratio = __fmul_rn(s_old, inv);
    // a piece is written when it holds a new position, or an earlier one whose scale grew
    uint32_t fresh[4], old[4];   // V: the same in every word
    bool any_fresh = false, any_old = false, whole = true;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        fresh[k] = piece_mask<V>(lane, V ? 0 : k, first, m);
        old[k] = piece_mask<V>(lane, V ? 0 : k, 0, first);
        any_fresh |= fresh[k] != 0;
        any_old |= old[k] != 0;
        whole &= fresh[k] == 0xffffffffu;
    }
    if (any_fresh || (grew && any_old)) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            uint4* pc = reinterpret_cast<uint4*>(code + c * 512);
            const float* v = val[c];
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
                w[k] = V ? encode4<E4M3>(__fmul_rn(v[k], inv), __fmul_rn(v[4 + k], inv), __fmul_rn(v[8 + k], inv),
                                         __fmul_rn(v[12 + k], inv))
                         : encode4<E4M3>(__fmul_rn(v[4 * k], inv), __fmul_rn(v[4 * k + 1], inv),
                                         __fmul_rn(v[4 * k + 2], inv), __fmul_rn(v[4 * k + 3], inv));
            if (!whole) {
                const uint4 q = *pc;
                const uint32_t was[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t x = was[k];
                    if (grew && old[k]) {
                        float f[4];
                        decode4<E4M3>(x, f);
                        x = encode4<E4M3>(__fmul_rn(f[0], ratio), __fmul_rn(f[1], ratio), __fmul_rn(f[2], ratio),
                                          __fmul_rn(f[3], ratio));
                        x = (x & old[k]) | (was[k] & ~old[k]);
                    }
                    w[k] = (w[k] & fresh[k]) | (x & ~fresh[k]);
                }
            }
            *pc = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __syncwarp();
    if (lane == 0) *sp = s;
}

template <int HD, int DT, bool E4M3>
__global__ void __launch_bounds__(kAppendWarps * 32) kv8_append_kernel(const AppendArgs a) {
    const int lane = threadIdx.x & 31;
    const Kv8Tables& t = a.t;
    const int nrows = min(t.meta->rows, a.rows), units = t.meta->units;
    const long long total = (long long)units * a.kv_heads * 2;
    for (long long w = (long long)blockIdx.x * kAppendWarps + (threadIdx.x >> 5); w < total;
         w += (long long)gridDim.x * kAppendWarps) {
        const int h = (int)((w >> 1) % a.kv_heads), u = (int)((w >> 1) / a.kv_heads);
        const int r0 = t.unit_row[u];
        if (r0 >= nrows) continue;
        const int b = t.row_seq[r0], slot0 = t.slot[r0];
        const int first = slot0 % kKv8Block;            // first new position of the block
        const int m = min(kKv8Block - first, min(t.row_start[b + 1], nrows) - r0);
        const size_t ph = (size_t)(slot0 / kPageSize) * a.kv_heads + h;
        const int blk = slot0 % kPageSize / kKv8Block;
        const size_t off = ph * (kPageSize * HD) + (size_t)blk * (kKv8Block * HD) + lane * 16;
        const size_t sc = ph * kKv8Sub + blk;
        if (w & 1)
            append_block<HD, DT, E4M3, true>(a.v, (size_t)r0 * a.ldv + (size_t)h * HD, a.ldv, a.vec, first, m,
                                             a.vc + off, a.vs + sc, lane);
        else
            append_block<HD, DT, E4M3, false>(a.k, (size_t)r0 * a.ldk + (size_t)h * HD, a.ldk, a.vec, first, m,
                                              a.kc + off, a.ks + sc, lane);
    }
}

// ---------------------------------------------------------------------------
// Gather: the values that the codes of every planned sequence stand for,
// packed [key][kv head][head_dim]. One warp per (16-position block, kv head,
// K or V); bound by the bytes written, at few blocks by the chain of loads before
// them (the block's sequence, page and scale).
// ---------------------------------------------------------------------------
struct GatherArgs {
    Kv8Tables t;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    void *ko, *vo;
    int keys, kv_heads, max_pages, vec;
};

template <int HD, int DT, bool E4M3, bool V>
__device__ __forceinline__ void gather_block(const uint8_t* code, float s, void* out, size_t at, size_t ld, int vec,
                                             int m, int lane) {
#pragma unroll
    for (int c = 0; c < HD / 32; c++) {
        const uint4 q = *reinterpret_cast<const uint4*>(code + c * 512);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        float v[4][4];
#pragma unroll
        for (int k = 0; k < 4; k++) decode4<E4M3>(w[k], v[k]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p = piece_pos<V>(lane, i);
            if (p >= m) continue;
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] = __fmul_rn(V ? v[j][i] : v[i][j], s);
            store4<DT>(out, at + (size_t)p * ld + c * 32 + piece_dim<V>(lane, i), vec, f);
        }
    }
}

template <int HD, int DT, bool E4M3>
__global__ void __launch_bounds__(kAppendWarps * 32) kv8_gather_kernel(const GatherArgs a) {
    const int lane = threadIdx.x & 31;
    const Kv8Tables& t = a.t;
    const int nseq = t.meta->seqs;
    const size_t ld = (size_t)a.kv_heads * HD;
    const long long total = (long long)t.meta->gblocks * a.kv_heads * 2;
    for (long long w = (long long)blockIdx.x * kAppendWarps + (threadIdx.x >> 5); w < total;
         w += (long long)gridDim.x * kAppendWarps) {
        const int h = (int)((w >> 1) % a.kv_heads), g = (int)((w >> 1) / a.kv_heads);
        // cached loads: the starts are an earlier kernel's (past L1 the search took most of the time)
        const int b = find_seq_by(nseq, g, [&](int k) { return t.gblk_start[k]; });
        const int blk = g - t.gblk_start[b];
        const int k0 = t.kv_start[b] + blk * kKv8Block;
        const int m = min(kKv8Block, min(t.kv_start[b + 1], a.keys) - k0);
        if (m <= 0) continue;
        const size_t ph = (size_t)t.block_table[(size_t)b * a.max_pages + blk / kKv8Sub] * a.kv_heads + h;
        const size_t off = ph * (kPageSize * HD) + (size_t)(blk % kKv8Sub) * (kKv8Block * HD) + lane * 16;
        const size_t sc = ph * kKv8Sub + blk % kKv8Sub;
        const size_t at = (size_t)k0 * ld + (size_t)h * HD;
        if (w & 1)
            gather_block<HD, DT, E4M3, true>(a.vc + off, a.vs[sc], a.vo, at, ld, a.vec, m, lane);
        else
            gather_block<HD, DT, E4M3, false>(a.kc + off, a.ks[sc], a.ko, at, ld, a.vec, m, lane);
    }
}

int elem_size(int dtype) { return dtype == FL_F32 ? 4 : 2; }

// Calls f<HD, DT, E4M3>() for the handle's configuration.
template <template <int, int, bool> class F, typename... A>
cudaError_t dispatch(const fl_kv8_config_t& c, A... args) {
#define FL_KV8_HD(HD)                                                                                   \
    if (c.head_dim == HD) {                                                                             \
        if (c.type == FL_KV8_E4M3) {                                                                    \
            if (c.dtype == FL_F32) return F<HD, FL_F32, true>::run(args...);                            \
            if (c.dtype == FL_F16) return F<HD, FL_F16, true>::run(args...);                            \
            return F<HD, FL_BF16, true>::run(args...);                                                  \
        }                                                                                               \
        if (c.dtype == FL_F32) return F<HD, FL_F32, false>::run(args...);                               \
        if (c.dtype == FL_F16) return F<HD, FL_F16, false>::run(args...);                               \
        return F<HD, FL_BF16, false>::run(args...);                                                     \
    }
    FL_KV8_HD(32)
    FL_KV8_HD(64)
    FL_KV8_HD(96)
    FL_KV8_HD(128)
#undef FL_KV8_HD
    return cudaErrorInvalidValue;
}

template <int HD, int DT, bool E4M3>
struct RunAppend {
    static cudaError_t run(const AppendArgs* a, int grid, cudaStream_t s) {
        kv8_append_kernel<HD, DT, E4M3><<<grid, kAppendWarps * 32, 0, s>>>(*a);
        return cudaGetLastError();
    }
};
template <int HD, int DT, bool E4M3>
struct RunGather {
    static cudaError_t run(const GatherArgs* a, int grid, cudaStream_t s) {
        kv8_gather_kernel<HD, DT, E4M3><<<grid, kAppendWarps * 32, 0, s>>>(*a);
        return cudaGetLastError();
    }
};

// Common checks of the calls on a handle.
int check_handle(const fl_kv8* h, const char* what) {
    if (!h) return set_error(FL_E_INVAL, std::string(what) + ": handle is NULL");
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev != h->device) {
        cudaGetLastError();
        return set_error(FL_E_STATE, std::string(what) + ": the cache lives on another device than the current one");
    }
    return FL_OK;
}

int check_layer(const fl_kv8* h, int layer, const char* what) {
    FL_CHECK(check_handle(h, what));
    if (layer < 0 || layer >= h->c.layers) return set_error(FL_E_INVAL, std::string(what) + ": no such layer");
    if (h->nseq == 0) return set_error(FL_E_STATE, std::string(what) + ": no plan yet (fl_kv8_plan)");
    return FL_OK;
}

// The capture that a stream's calls go into, 0: none.
unsigned long long capture_of(cudaStream_t s) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(s, &st, &id) != cudaSuccess) {   // the legacy stream while another one is captured
        cudaGetLastError();
        return 0;
    }
    return st == cudaStreamCaptureStatusActive ? id : 0;
}

bool aligned(const void* p, size_t ld, int es) { return ((uintptr_t)p & 15) == 0 && ld * es % 16 == 0; }

template <typename T>
int alloc(fl_kv8* h, T** p, size_t count, bool zero) {
    void* q = nullptr;
    const size_t bytes = std::max<size_t>(count * sizeof(T), 16);
    FL_CHECK_CUDA(cudaMalloc(&q, bytes));
    h->bufs.push_back(q);
    if (zero) FL_CHECK_CUDA(cudaMemset(q, 0, bytes));
    *p = (T*)q;
    return FL_OK;
}

int create(fl_kv8* h) {
    const fl_kv8_config_t& c = h->c;
    h->max_pages = (c.max_ctx + kPageSize - 1) / kPageSize;
    h->group = c.heads / c.kv_heads;
    h->tile_rows = c.dtype == FL_F32 ? 8 : 16;
    cudaDeviceGetAttribute(&h->sms, cudaDevAttrMultiProcessorCount, h->device);
    h->parts[0] = h->sms * kv8_attention_occupancy(c.head_dim, c.type, c.dtype);
    FL_CHECK_CUDA(kv8_prefill_prepare(c.head_dim, c.type, c.dtype));
    h->parts[1] = h->sms;   // one CTA holds an SM's TMEM
    const size_t S = c.max_seqs, R = c.max_rows, kvb = (size_t)c.pages * c.kv_heads * kPageSize * c.head_dim;
    h->k.resize(c.layers);
    h->v.resize(c.layers);
    h->ks.resize(c.layers);
    h->vs.resize(c.layers);
    for (int l = 0; l < c.layers; l++) {
        FL_CHECK(alloc(h, &h->k[l], kvb, true));
        FL_CHECK(alloc(h, &h->v[l], kvb, true));
        FL_CHECK(alloc(h, &h->ks[l], (size_t)c.pages * c.kv_heads * kKv8Sub, true));
        FL_CHECK(alloc(h, &h->vs[l], (size_t)c.pages * c.kv_heads * kKv8Sub, true));
    }
    Kv8Tables& t = h->t;
    FL_CHECK(alloc(h, &t.block_table, S * h->max_pages, true));
    FL_CHECK(alloc(h, &t.held, S, true));
    FL_CHECK(alloc(h, &t.free_pages, c.pages, true));
    FL_CHECK(alloc(h, &t.n_free, 1, true));
    FL_CHECK(alloc(h, &t.status, 1, true));
    FL_CHECK(alloc(h, &t.slot, R, true));
    FL_CHECK(alloc(h, &t.pos, R, true));
    FL_CHECK(alloc(h, &t.row_seq, R, true));
    FL_CHECK(alloc(h, &t.unit_row, R, true));
    for (int** p : {&t.row_start, &t.kv_start, &t.take_start, &t.rel_start, &t.unit_start, &t.gblk_start, &t.ctx})
        FL_CHECK(alloc(h, p, S + 1, true));
    for (int i = 0; i < 2; i++) {
        FL_CHECK(alloc(h, &t.tile_start[i], S + 1, true));
        FL_CHECK(alloc(h, &t.work_start[i], S + 1, true));
    }
    FL_CHECK(alloc(h, &t.meta, 1, true));
    // a part begins inside a tile at most, and ends inside one
    for (int i = 0; i < 2; i++) {
        const size_t rows = (size_t)2 * h->parts[i] * (i ? kKv8Long : h->tile_rows);
        FL_CHECK(alloc(h, &h->part[i], rows * c.head_dim, false));
        FL_CHECK(alloc(h, &h->part_ml[i], rows, false));
        FL_CHECK(alloc(h, &h->part_cnt[i], h->parts[i], true));
    }
    FL_CHECK(alloc(h, &h->fold, (size_t)h->parts[1] * (c.head_dim / 4) * kKv8Long, false));
    kv8_reset_kernel<<<64, 256>>>(t, c.pages, c.max_seqs);
    FL_CHECK_CUDA(cudaGetLastError());
    FL_CHECK_CUDA(cudaDeviceSynchronize());
    return FL_OK;
}

}  // namespace

}  // namespace fl

using namespace fl;

FL_API fl_kv8_t* fl_kv8_create(const fl_kv8_config_t* cfg, int device) {
    if (!cfg) {
        set_error(FL_E_INVAL, "kv8_create: config is NULL");
        return nullptr;
    }
    const fl_kv8_config_t c = *cfg;
    const char* bad = nullptr;
    if (c.layers < 1 || c.heads < 1 || c.kv_heads < 1 || c.pages < 1 || c.max_seqs < 1 || c.max_rows < 1 || c.max_ctx < 1)
        bad = "kv8_create: every size must be at least 1";
    else if (c.heads % c.kv_heads)
        bad = "kv8_create: heads must be a multiple of kv_heads";
    else if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 96 && c.head_dim != 128)
        bad = "kv8_create: head_dim must be 32, 64, 96 or 128";
    else if (c.type != FL_KV8_INT8 && c.type != FL_KV8_E4M3)
        bad = "kv8_create: type must be FL_KV8_INT8 or FL_KV8_E4M3";
    else if (c.dtype != FL_F32 && c.dtype != FL_F16 && c.dtype != FL_BF16)
        bad = "kv8_create: dtype must be FL_F32, FL_F16 or FL_BF16";
    else if (c.layers > 4096 || c.heads > 4096 || c.max_seqs > 65536 || c.pages > (1 << 24) || c.max_rows > (1 << 24) ||
             c.max_ctx > (1 << 28) || (long long)c.max_rows * (c.heads / c.kv_heads) > (1 << 28))
        bad = "kv8_create: a size is beyond its limit (4096 layers or heads, 65536 sequences, 2^24 pages or rows, "
              "2^28 positions)";
    if (bad) {
        set_error(FL_E_INVAL, bad);
        return nullptr;
    }
    if (ensure_device() != FL_OK) return nullptr;
    int prev = 0, n = 0;
    if (cudaGetDevice(&prev) != cudaSuccess || cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n) {
        cudaGetLastError();
        set_error(FL_E_INVAL, "kv8_create: no such device");
        return nullptr;
    }
    fl_kv8* h = new (std::nothrow) fl_kv8;
    if (!h) {
        set_error(FL_E_NOMEM, "kv8_create: host allocation");
        return nullptr;
    }
    h->c = c;
    h->device = device;
    int rc = FL_E_NOMEM;
    if (cudaSetDevice(device) == cudaSuccess) {
        try {
            rc = create(h);
        } catch (...) {   // host allocation; no exception leaves a C entry
            rc = set_error(FL_E_NOMEM, "kv8_create: host allocation");
        }
    }
    if (rc != FL_OK) {
        fl_kv8_destroy(h);
        h = nullptr;
    }
    cudaSetDevice(prev);
    return h;
}

FL_API void fl_kv8_destroy(fl_kv8_t* h) {
    if (!h) return;
    int prev = 0;
    cudaGetDevice(&prev);
    cudaSetDevice(h->device);
    for (void* p : h->bufs) cudaFree(p);
    cudaSetDevice(prev);
    delete h;
}

FL_API int fl_kv8_tables(const fl_kv8_t* h, fl_kv8_tables_t* out) {
    if (!h || !out) return set_error(FL_E_INVAL, "kv8_tables: NULL argument");
    const Kv8Tables& t = h->t;
    *out = fl_kv8_tables_t{t.block_table, t.held, t.free_pages, t.n_free, t.row_start, t.kv_start,
                           t.slot, t.pos, t.row_seq, t.status, h->max_pages};
    return FL_OK;
}

FL_API int fl_kv8_plan(fl_kv8_t* h, const int* ctx_len, const int* new_len, int nseq, int max_new, void* stream) {
    FL_CHECK(check_handle(h, "kv8_plan"));
    if (!ctx_len || !new_len) return set_error(FL_E_INVAL, "kv8_plan: NULL lengths");
    if (nseq < 1 || nseq > h->c.max_seqs) return set_error(FL_E_INVAL, "kv8_plan: nseq must be 1 .. max_seqs");
    if (max_new < 1) return set_error(FL_E_INVAL, "kv8_plan: max_new must be at least 1");
    if (((uintptr_t)ctx_len | (uintptr_t)new_len) % sizeof(int))
        return set_error(FL_E_INVAL, "kv8_plan: lengths are not aligned to their type");
    FL_CHECK(check_device_ptr(ctx_len, "kv8_plan: ctx_len"));
    FL_CHECK(check_device_ptr(new_len, "kv8_plan: new_len"));
    cudaStream_t s = stream ? (cudaStream_t)stream : device_stream();
    PlanArgs a = {};
    a.ctx = ctx_len;
    a.nw = new_len;
    a.t = h->t;
    a.nseq = nseq;
    a.max_new = std::min(max_new, h->c.max_rows);
    a.max_pages = h->max_pages;
    a.max_rows = h->c.max_rows;
    a.group = h->group;
    a.tile_rows = h->tile_rows;
    a.long_min = long_min(h);
    // one CTA while its threads hold the rows; eight (a portable cluster) beyond
    const long long rows = std::min<long long>((long long)nseq * a.max_new, h->c.max_rows);
    const bool small = nseq <= 256 && rows <= 1024;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = rows > 4096 ? 8 : 1;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(at[0].val.clusterDim.x);
    cfg.blockDim = dim3(small ? 256 : 1024);
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = rows > 4096 ? 1 : 0;
    FL_CHECK_CUDA(cudaLaunchKernelEx(&cfg, small ? kv8_plan_kernel<256> : kv8_plan_kernel<1024>, a));
    h->nseq = nseq;
    h->max_new = a.max_new;
    h->plan_capture = capture_of(s);
    if (h->plan_capture) h->captured_max_new = std::max(h->captured_max_new, a.max_new);
    return FL_OK;
}

FL_API int fl_kv8_append(fl_kv8_t* h, int layer, const void* k, const void* v, int rows, size_t ldk, size_t ldv,
                         void* stream) {
    FL_CHECK(check_layer(h, layer, "kv8_append"));
    if (rows < 0) return set_error(FL_E_INVAL, "kv8_append: rows is negative");
    if (rows == 0) return FL_OK;
    const size_t w = (size_t)h->c.kv_heads * h->c.head_dim;
    if (!k || !v) return set_error(FL_E_INVAL, "kv8_append: NULL rows");
    if (rows > 1 && (ldk < w || ldv < w)) return set_error(FL_E_INVAL, "kv8_append: a row stride is below kv_heads * head_dim");
    const int es = elem_size(h->c.dtype);
    if ((uintptr_t)k % es || (uintptr_t)v % es) return set_error(FL_E_INVAL, "kv8_append: rows are not aligned to their type");
    FL_CHECK(check_device_ptr(k, "kv8_append: k"));
    FL_CHECK(check_device_ptr(v, "kv8_append: v"));
    cudaStream_t s = stream ? (cudaStream_t)stream : device_stream();
    AppendArgs a = {};
    a.t = h->t;
    a.k = k;
    a.v = v;
    a.ldk = ldk;
    a.ldv = ldv;
    a.kc = h->k[layer];
    a.vc = h->v[layer];
    a.ks = h->ks[layer];
    a.vs = h->vs[layer];
    a.rows = rows;
    a.kv_heads = h->c.kv_heads;
    a.vec = aligned(k, ldk, es) && aligned(v, ldv, es);
    const long long units = std::min<long long>(rows, rows / kKv8Block + 2ll * h->nseq) * a.kv_heads * 2;
    const int grid = (int)std::min<long long>((units + kAppendWarps - 1) / kAppendWarps, (long long)h->sms * 32);
    FL_CHECK_CUDA((dispatch<RunAppend>(h->c, &a, grid, s)));
    return FL_OK;
}

FL_API int fl_kv8_gather(fl_kv8_t* h, int layer, void* k, void* v, int keys, void* stream) {
    FL_CHECK(check_layer(h, layer, "kv8_gather"));
    if (keys < 0) return set_error(FL_E_INVAL, "kv8_gather: keys is negative");
    if (keys == 0) return FL_OK;
    if (!k || !v) return set_error(FL_E_INVAL, "kv8_gather: NULL outputs");
    const int es = elem_size(h->c.dtype);
    if ((uintptr_t)k % es || (uintptr_t)v % es) return set_error(FL_E_INVAL, "kv8_gather: outputs are not aligned to their type");
    FL_CHECK(check_device_ptr(k, "kv8_gather: k"));
    FL_CHECK(check_device_ptr(v, "kv8_gather: v"));
    cudaStream_t s = stream ? (cudaStream_t)stream : device_stream();
    GatherArgs a = {};
    a.t = h->t;
    a.kc = h->k[layer];
    a.vc = h->v[layer];
    a.ks = h->ks[layer];
    a.vs = h->vs[layer];
    a.ko = k;
    a.vo = v;
    a.keys = keys;
    a.kv_heads = h->c.kv_heads;
    a.max_pages = h->max_pages;
    a.vec = aligned(k, 16, es) && aligned(v, 16, es);
    const long long units = ((long long)keys / kKv8Block + h->nseq) * a.kv_heads * 2;
    const int grid = (int)std::min<long long>((units + kAppendWarps - 1) / kAppendWarps, (long long)h->sms * 32);
    FL_CHECK_CUDA((dispatch<RunGather>(h->c, &a, grid, s)));
    return FL_OK;
}

namespace {

// How a call's bounded waits behave: their limit, and a CTA that gives up (fl_kv8.h).
struct Waits {
    long long clocks = kKv8WaitClocks;
    int fail_cta = 0, fail_at = 0;
};

int attention(fl_kv8_t* h, int layer, const void* q, void* out, int rows, size_t ldq, size_t ldo, float scale,
              const uint8_t* mask, int ldm, const Waits& wait, void* stream) {
    FL_CHECK(check_layer(h, layer, "kv8_attention"));
    if (rows < 0) return set_error(FL_E_INVAL, "kv8_attention: rows is negative");
    if (rows == 0) return FL_OK;
    const size_t w = (size_t)h->c.heads * h->c.head_dim;
    if (!q || !out) return set_error(FL_E_INVAL, "kv8_attention: NULL rows");
    if (rows > 1 && (ldq < w || ldo < w)) return set_error(FL_E_INVAL, "kv8_attention: a row stride is below heads * head_dim");
    if (!(scale == scale) || scale - scale != 0.0f) return set_error(FL_E_INVAL, "kv8_attention: scale is not finite");
    const int es = elem_size(h->c.dtype);
    if ((uintptr_t)q % es || (uintptr_t)out % es)
        return set_error(FL_E_INVAL, "kv8_attention: rows are not aligned to their type");
    if (mask && ldm < h->max_new) return set_error(FL_E_INVAL, "kv8_attention: mask rows are shorter than max_new");
    FL_CHECK(check_device_ptr(q, "kv8_attention: q"));
    FL_CHECK(check_device_ptr(out, "kv8_attention: out"));
    if (mask) FL_CHECK(check_device_ptr(mask, "kv8_attention: mask"));
    cudaStream_t s = stream ? (cudaStream_t)stream : device_stream();
    Kv8AttnParams p = {};
    p.k = h->k[layer];
    p.v = h->v[layer];
    p.ks = h->ks[layer];
    p.vs = h->vs[layer];
    p.t = h->t;
    p.max_pages = h->max_pages;
    p.heads = h->c.heads;
    p.kv_heads = h->c.kv_heads;
    p.group = h->group;
    p.head_dim = h->c.head_dim;
    p.type = h->c.type;
    p.dtype = h->c.dtype;
    p.q = q;
    p.out = out;
    p.ldq = ldq;
    p.ldo = ldo;
    p.rows = rows;
    p.scale = scale * 1.4426950408889634f;
    p.mask = mask;
    p.ldm = ldm;
    Kv8Tiles tl[2];
    for (int i = 0; i < 2; i++)
        tl[i] = Kv8Tiles{i, h->t.tile_start[i], h->t.work_start[i], h->part[i], h->part_ml[i], h->part_cnt[i],
                         h->fold, wait.clocks, wait.fail_cta, wait.fail_at};
    FL_CHECK_CUDA(launch_kv8_attention(p, tl[0], h->parts[0], s));
    // The plan that this call will find may be a replayed one, unless both are in one capture
    const bool own_plan = h->plan_capture && h->plan_capture == capture_of(s);
    const long long max_new = own_plan ? h->max_new : std::max(h->max_new, h->captured_max_new);
    if (max_new * h->group >= long_min(h)) FL_CHECK_CUDA(launch_kv8_prefill(p, tl[1], h->parts[1], s));
    return FL_OK;
}

}  // namespace

FL_API int fl_kv8_attention(fl_kv8_t* h, int layer, const void* q, void* out, int rows, size_t ldq, size_t ldo,
                            float scale, const uint8_t* mask, int ldm, void* stream) {
    return attention(h, layer, q, out, rows, ldq, ldo, scale, mask, ldm, Waits{}, stream);
}

FL_API int fl_kv8_wait_timeout_check(fl_kv8_t* h, int layer, const void* q, void* out, int rows, size_t ldq, size_t ldo,
                                     float scale, int cta, int at, void* stream) {
    if (cta < 0 || at < 1) return set_error(FL_E_INVAL, "kv8_wait_timeout_check: cta or at is out of range");
    // every other wait of that CTA runs out, too: a tenth of a second each
    return attention(h, layer, q, out, rows, ldq, ldo, scale, nullptr, 0, Waits{200000000ll, cta, at}, stream);
}
