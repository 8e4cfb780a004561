// The integer sampling weight that every device sampler uses (the rule is
// stated in include/speculative.h and at the head of sample_ops.cu).
#pragma once

#include <stdint.h>

namespace fl {

constexpr uint32_t kOne = 1u << 24;

// E = trunc(e^x * 2^24) for x <= 0, 0 below x = -17 and for NaN: e^x by
// Cody-Waite reduction by ln 2 and a degree-7 Taylor polynomial in Horner
// form, each step correctly rounded, then the exact scale by 2^(k + 24).
// e^-17 2^24 = 0.69, so everything below -16.64 gives 0 by itself and a clamp at
// -18 serves for the cut. k and its float come from the sum with 1.5 2^23 + 24,
// whose low bits are k + 24 (an even offset keeps the rounding to even, and the
// constant's own bits leave the word in the shift), so that the truncation is the
// only conversion: those run at a quarter of the other instructions' rate.
__device__ __forceinline__ uint32_t sample_weight(float x) {
    x = fmaxf(x, -18.0f);
    const float magic = __fadd_rn(__fmul_rn(x, 1.442695f), 12582936.0f);
    const float kf = __fsub_rn(magic, 12582936.0f);
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
    // k in [-26, 0]: p 2^(k + 24) is a normal float, at most 2^24 (p <= 1 at k = 0)
    return __float2uint_rz(__int_as_float(__float_as_int(p) + (__float_as_int(magic) << 23)));
}

}  // namespace fl
