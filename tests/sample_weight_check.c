/* The order of the sampling weights (fl_sample.cuh, the same operations in
 * host arithmetic) over every float from -18.5 up to -2^-40 and zero: prints
 * by how much the weight of a float lies below that of a smaller one at most,
 * for how many floats it does, and the smallest and the largest weight of such
 * a pair. */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

static float from_bits(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static uint32_t bits(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }

static uint32_t weight(float x) {
    x = fmaxf(x, -18.0f);
    const float prod = x * 1.442695f;
    const float magic = prod + 12582936.0f;
    const float kf = magic - 12582936.0f;
    float r = fmaf(-kf, 0.693145751953125f, x);
    r = fmaf(-kf, 1.4286068e-06f, r);
    float p = 0.0001984127f;
    p = fmaf(p, r, 0.0013888889f);
    p = fmaf(p, r, 0.008333334f);
    p = fmaf(p, r, 0.041666668f);
    p = fmaf(p, r, 0.16666667f);
    p = fmaf(p, r, 0.5f);
    p = fmaf(p, r, 1.0f);
    p = fmaf(p, r, 1.0f);
    return (uint32_t)from_bits(bits(p) + (bits(magic) << 23));
}

int main(void) {
    uint32_t top = 0, below = 0, lo = 0xffffffffu, hi = 0;
    long n = 0;
    for (uint32_t u = bits(-18.5f);; u--) {
        if (u < bits(-0x1p-40f)) u = bits(-0.0f);
        const uint32_t e = weight(from_bits(u));
        if (e < top) {
            n++;
            if (top - e > below) below = top - e;
            if (e < lo) lo = e;
            if (top > hi) hi = top;
        } else {
            top = e;
        }
        if (u == bits(-0.0f)) break;
    }
    printf("below %u floats %ld weights %u to %u largest %u\n", below, n, lo, hi, top);
    return 0;
}
