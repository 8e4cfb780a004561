// The integer sampling weight that every device sampler uses (the rule is
// stated in include/speculative.h and at the head of sample_ops.cu).
#pragma once

#include <stdint.h>

namespace fl {

constexpr uint32_t kOne = 1u << 24;

// E = trunc(e^x * 2^24) for x <= 0, 0 below x = -17: e^x by Cody-Waite
// reduction by ln 2 and a degree-7 Taylor polynomial in Horner form, each step
// correctly rounded, then the exact scale by 2^(k + 24).
__device__ __forceinline__ uint32_t sample_weight(float x) {
    if (!(x >= -17.0f)) return 0u;
    const float kf = rintf(__fmul_rn(x, 1.442695f));
    float r = __fmaf_rn(-kf, 0.693145751953125f, x);
    r = __fmaf_rn(-kf, 1.4286068e-06f, r);
    float p = 0.0001984127f;
    p = __fmaf_rn(p, r, 0.0013888889f);
    p = __fmaf_rn(p, r, 0.008333334f);
    p = __fmaf_rn(p, r, 0.041666668f);
    p = __fmaf_rn(p, r, 0.16666667f);
    p = __fmaf_rn(p, r, 0.5f);
    p = __fmaf_rn(p, r, 1.0f);
    p = __fmaf_rn(p, r, 1.0f);
    const int e = 127 + 24 + (int)kf;  // 2^(k + 24), k in [-25, 0]: a normal float
    const uint32_t E = __float2uint_rz(__fmul_rn(p, __int_as_float(e << 23)));
    return E > kOne ? kOne : E;
}

}  // namespace fl
