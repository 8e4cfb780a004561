// Conversions of the 8-bit KV cache: 4-element loads and stores of the
// activation types, power-of-two scales, codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "fl_cuda.h"

namespace fl {

// Four consecutive elements at index i (a multiple of 4) as floats; vec: the
// base and the strides allow one load.
template <int DT>
__device__ __forceinline__ void load4(const void* x, size_t i, int vec, float (&f)[4]) {
    if constexpr (DT == FL_F32) {
        const float* p = static_cast<const float*>(x) + i;
        if (vec) {
            const float4 v = *reinterpret_cast<const float4*>(p);
            f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] = p[j];
        }
    } else if constexpr (DT == FL_F16) {
        const __half* p = static_cast<const __half*>(x) + i;
        if (vec) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
            const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
            f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] = __half2float(p[j]);
        }
    } else {
        const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(x) + i;
        if (vec) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
            f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] = __bfloat162float(p[j]);
        }
    }
}

template <int DT>
__device__ __forceinline__ void store4(void* x, size_t i, int vec, const float (&f)[4]) {
    if constexpr (DT == FL_F32) {
        float* p = static_cast<float*>(x) + i;
        if (vec) {
            *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) p[j] = f[j];
        }
    } else if constexpr (DT == FL_F16) {
        __half* p = static_cast<__half*>(x) + i;
        const __half2 a = __floats2half2_rn(f[0], f[1]), b = __floats2half2_rn(f[2], f[3]);
        if (vec) {
            *reinterpret_cast<uint2*>(p) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
            p[0] = __low2half(a); p[1] = __high2half(a); p[2] = __low2half(b); p[3] = __high2half(b);
        }
    } else {
        __nv_bfloat16* p = static_cast<__nv_bfloat16*>(x) + i;
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
        if (vec) {
            *reinterpret_cast<uint2*>(p) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
            p[0] = __low2bfloat16(a); p[1] = __high2bfloat16(a); p[2] = __low2bfloat16(b); p[3] = __high2bfloat16(b);
        }
    }
}

// The smallest power of two s = 2^e, e >= -100, with amax <= top * s (top 127
// or 448): amax = m 2^x with 1 <= m < 2, 127 = (127/64) 2^6, 448 = 1.75 2^8.
// From the float's bits, so exact; subnormals have x < -126 and end at -100.
template <bool E4M3>
__device__ __forceinline__ float pow2_scale(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int x = (int)(b >> 23) - 127;
    const uint32_t frac = b & 0x7fffffu;
    const int e = E4M3 ? x - 8 + (frac > 0x600000u) : x - 6 + (frac > 0x7e0000u);
    return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}
// 1 / s of a power of two within 2^-126 .. 2^126.
__device__ __forceinline__ float pow2_inv(float s) {
    return __uint_as_float((254u << 23) - __float_as_uint(s));
}

// Four codes of y = x / scale in a word, rounded to nearest even, beyond the
// largest code to it (infinities too), NaN to zero. INT8 codes are stored plus
// 128: y + 1.5 2^23 + 128 is y rounded, plus 128, in the low byte.
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    float y[4] = {a, b, c, d};
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = y[i] != y[i] ? 0.0f : y[i];
    if constexpr (E4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(y[i], -127.0f), 127.0f), 12583040.0f));
        return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    }
}
// The four values of a word's codes.
template <bool E4M3>
__device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
    if constexpr (E4M3) {
        const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3)));
        const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    } else {
        // byte u under 0x4b0000: the float 2^23 + u
#pragma unroll
        for (int i = 0; i < 4; i++)
            f[i] = __fsub_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)), 8388736.0f);
    }
}

}  // namespace fl
