// One token per logits row from given uniform numbers (sm_100a): temperature,
// top-k, min-p and top-p on the integer weights of the library's sampling rule
// (fl_sample.cuh), so every sum is exact and the draw does not depend on the
// order of any reduction. The rule is stated at fl_cuda_sample in
// include/fl_cuda.h.
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
constexpr int kT = 1024, kW = kT / 32;

struct SampleArgs {
    const void* logits;
    size_t ld;
    int V;
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* tokens;
};

// Logit i as the rule reads it: NaN counts as -inf, +inf as the largest float, -0 as 0.
template <int DT>
__device__ __forceinline__ float logit(const void* l, int i) {
    float x;
    if constexpr (DT == FL_F32) x = static_cast<const float*>(l)[i];
    else if constexpr (DT == FL_F16) x = __half2float(static_cast<const __half*>(l)[i]);
    else x = __bfloat162float(static_cast<const __nv_bfloat16*>(l)[i]);
    return x != x ? -INFINITY : fminf(x, FLT_MAX) + 0.0f;
}
// Orders floats as unsigned integers.
__device__ __forceinline__ uint32_t sortable(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ unsigned long long bsum(unsigned long long v, unsigned long long* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long t = red[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}
__device__ __forceinline__ unsigned long long bmax64(unsigned long long v, unsigned long long* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long t = red[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
    return t;
}

// trunc(p 2^24) within [0, 2^24]; 0 for NaN.
__device__ __forceinline__ uint32_t fixed24(float p) {
    return __float2uint_rz(__fmul_rn(fminf(fmaxf(p, 0.0f), 1.0f), 16777216.0f));
}

template <int DT>
__global__ void __launch_bounds__(kT) sample_rows_kernel(const SampleArgs a) {
    __shared__ unsigned long long red[kW];
    __shared__ int pick_s;
    const int r = blockIdx.x, V = a.V;
    const size_t es = DT == FL_F32 ? 4 : 2;
    const void* l = static_cast<const char*>(a.logits) + (size_t)r * a.ld * es;
    unsigned long long key = 0;
    for (int i = threadIdx.x; i < V; i += kT) key = max(key, argmax_key(logit<DT>(l, i), i));
    key = bmax64(key, red);
    const float mx = argmax_key_value(key);
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    if (mx == -INFINITY || !(T > 0.0f)) {
        if (threadIdx.x == 0) a.tokens[r] = mx == -INFINITY ? -1 : argmax_key_index(key);
        return;
    }
    // lowest key kept by top-k, and the last index kept among its equals
    uint32_t klo = 0;
    int ilast = V - 1;
    const int k = a.top_k ? a.top_k[r] : 0;
    if (k > 0 && k < V) {
        uint32_t hi = 0xffffffffu;   // largest key with at least k logits at or above it
        while (hi - klo > 1u) {
            const uint32_t mid = klo + (hi - klo) / 2u;
            unsigned long long c = 0;
            for (int i = threadIdx.x; i < V; i += kT) c += sortable(logit<DT>(l, i)) >= mid;
            if (bsum(c, red) >= (unsigned long long)k) klo = mid; else hi = mid;
        }
        unsigned long long above = 0;
        for (int i = threadIdx.x; i < V; i += kT) above += sortable(logit<DT>(l, i)) > klo;
        const unsigned long long ties = (unsigned long long)k - bsum(above, red);
        int lo = -1, up = V - 1;     // smallest index with `ties` equals at or before it
        while (up - lo > 1) {
            const int mid = lo + (up - lo) / 2;
            unsigned long long c = 0;
            for (int i = threadIdx.x; i <= mid; i += kT) c += sortable(logit<DT>(l, i)) == klo;
            if (bsum(c, red) >= ties) up = mid; else lo = mid;
        }
        ilast = up;
    }
    auto weight = [&](int i) -> uint32_t {
        const float x = logit<DT>(l, i);
        const uint32_t s = sortable(x);
        if (s < klo || (s == klo && i > ilast)) return 0u;
        return sample_weight(__fdiv_rn(__fsub_rn(x, mx), T));
    };
    uint32_t lo = max(1u, a.min_p ? fixed24(a.min_p[r]) : 0u);
    const float tp = a.top_p ? a.top_p[r] : 1.0f;
    if (tp < 1.0f) {
        unsigned long long z = 0;
        for (int i = threadIdx.x; i < V; i += kT) z += weight(i);
        z = bsum(z, red);
        const u128 need = (u128)max(1u, fixed24(tp)) * z;
        uint32_t b = 1u, hi = kOne + 1u;
        while (hi - b > 1u) {
            const uint32_t mid = b + (hi - b) / 2u;
            unsigned long long m = 0;
            for (int i = threadIdx.x; i < V; i += kT) {
                const uint32_t e = weight(i);
                m += e >= mid ? e : 0u;
            }
            if (((u128)bsum(m, red) << 24) >= need) b = mid; else hi = mid;
        }
        lo = max(lo, b);
    }
    // inverse CDF: thread t owns the contiguous chunk t
    const int C = (V + kT - 1) / kT;
    const int b0 = min(V, (int)threadIdx.x * C), b1 = min(V, b0 + C);
    unsigned long long local = 0;
    for (int i = b0; i < b1; i++) {
        const uint32_t e = weight(i);
        local += e >= lo ? e : 0u;
    }
    const unsigned long long total = bsum(local, red);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long inc = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) red[warp] = inc;
    if (threadIdx.x == 0) pick_s = V - 1;
    __syncthreads();
    unsigned long long c = inc - local;
    for (int w = 0; w < warp; w++) c += red[w];
    const uint32_t U = min(fixed24(a.u[r]), kOne - 1u);
    const unsigned long long tgt = (unsigned long long)(((u128)U * total) >> 24);
    if (c <= tgt && c + local > tgt) {
        for (int i = b0; i < b1; i++) {
            const uint32_t e = weight(i);
            c += e >= lo ? e : 0u;
            if (c > tgt) {
                pick_s = i;
                break;
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) a.tokens[r] = pick_s;
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
    if (V > (1 << 20)) return set_error(FL_E_INVAL, "sample: at most 2^20 tokens");
    if (rows > 1 && ld < (size_t)V) return set_error(FL_E_INVAL, "sample: the row stride is below V");
    if ((uintptr_t)logits % (dtype == FL_F32 ? 4 : 2))
        return set_error(FL_E_INVAL, "sample: logits are not aligned to their type");
    FL_CHECK(ensure_device());
    cudaStream_t s = stream ? (cudaStream_t)stream : device_stream();
    const SampleArgs a = {logits, ld, V, temperature, top_p, min_p, u, top_k, tokens};
    if (dtype == FL_F32) sample_rows_kernel<FL_F32><<<rows, kT, 0, s>>>(a);
    else if (dtype == FL_F16) sample_rows_kernel<FL_F16><<<rows, kT, 0, s>>>(a);
    else sample_rows_kernel<FL_BF16><<<rows, kT, 0, s>>>(a);
    FL_CHECK_CUDA(cudaGetLastError());
    return FL_OK;
}
