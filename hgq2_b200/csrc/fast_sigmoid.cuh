// The logistic function and its complement without an IEEE division.
#pragma once
#include <cuda_runtime.h>

namespace hgq {

// a = sigmoid(z) = 1 / (1 + e) with e = exp(-z), and c = 1 - a = e / (1 + e), each with a small relative error wherever it is a
// normal number (c is not the difference where a is near 1).  FULL (fp32 data): at most 12 x 2^-24; z is held in [-88, 100], where the
// two are 0 and 1; the exponential is 2^(-z log2 e) with what the product loses carried along: its rounding, and the part of log2 e
// below fp32 (2e-8, which would be 18 x 2^-24 of e at |z| = 80); the reciprocal's error is one ulp.  Otherwise (bf16 and fp16
// data): z has at most 11 bits and the outputs no more, the product's rounding (|z| 2^-24 of e) is far below both; a closed gate is
// 2^-126.  A NaN stays.
template <bool FULL>
__device__ __forceinline__ void sigmoid_pair(float z, float &a, float &c) {
    float e, r;
    if (FULL) {
        asm("max.NaN.f32 %0, %0, 0fC2B00000;" : "+f"(z));
        asm("min.NaN.f32 %0, %0, 0f42C80000;" : "+f"(z));
        const float t = z * -1.44269504088896341f;
        float lo = fmaf(z, -1.44269504088896341f, -t);
        lo = fmaf(z, -1.925962991126e-8f, lo);
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
        e = fmaf(e, lo * 0.693147180559945309f, e);
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
