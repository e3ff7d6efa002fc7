// The logistic function and its complement without an IEEE division.
#pragma once
#include <cuda_runtime.h>

namespace hgq {

// a = sigmoid(z) = 1 / (1 + e) with e = exp(-z), and c = 1 - a = e / (1 + e), each with a small relative error wherever it is a
// normal number (c is not the difference where a is near 1).
//
// FULL (fp32 data): counted at most 12 x 2^-24, measured 4.9.  z is held in [-88, 100], where the two are 0 and 1.
// e = 2^t exp(-z - t ln 2) with t near -z log2 e: ln 2 in two parts keeps what t loses by its own rounding and by that of log2 e (2e-8,
// which alone would be 18 x 2^-24 of e at |z| = 80).  The reciprocal's error is one ulp.
//
// Otherwise (bf16 and fp16 data; z may be any fp32 number): e = 2^t is off by about 1.2 |z| 2^-24 of it, at most 7e-6 up to |z| = 88 where
// the smaller of a and c vanishes, against 5e-4 and more that rounding the outputs to 11 bits costs; a closed gate is 2^-126.
//
// A NaN stays.
template <bool FULL>
__device__ __forceinline__ void sigmoid_pair(float z, float &a, float &c) {
    float e, r;
    if (FULL) {
        asm("max.NaN.f32 %0, %0, 0fC2B00000;" : "+f"(z));
        asm("min.NaN.f32 %0, %0, 0f42C80000;" : "+f"(z));
        const float t = z * -1.44269504088896341f;
        const float lo = fmaf(t, 1.90465429995776805e-9f, fmaf(t, -0.693147182464599609f, -z));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
        e = fmaf(e, lo, e);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
        a = r;
        c = z < 0.f ? 1.f - r : e * r;
    } else {
        float t = z * -1.44269504088896341f;
        asm("min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(t));  // 126
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
        a = r;
        c = e * r;
    }
}

}  // namespace hgq
