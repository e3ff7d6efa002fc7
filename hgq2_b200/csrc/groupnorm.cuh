// Pieces shared by the group normalisation kernels: vector accesses, activations, and the entry of the one-read kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fast_sigmoid.cuh"
#include "hgq_common.cuh"

namespace hgq {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float v, float &o) { o = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(float v, __half &o) { o = __float2half_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T *p, float (&f)[VEC]) {
    const Pack<T, VEC> q = *reinterpret_cast<const Pack<T, VEC> *>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_float(q.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T *p, const float (&f)[VEC]) {
    Pack<T, VEC> q;
#pragma unroll
    for (int i = 0; i < VEC; ++i) from_float(f[i], q.v[i]);
    *reinterpret_cast<Pack<T, VEC> *>(p) = q;
}

// act(u) for data of type T; ACT is HGQ_ACT_*
template <typename T, int ACT>
__device__ __forceinline__ float act_value(float u) {
    if (ACT == HGQ_ACT_RELU) return u < 0.f ? 0.f : u;  // a NaN stays
    if (ACT == HGQ_ACT_SILU) {
        float p, q;
        sigmoid_pair<sizeof(T) == 4>(u, p, q);
        return u * p;
    }
    if (ACT == HGQ_ACT_GELU) return 0.5f * u * (1.f + erff(u * 0.70710678118654752f));
    return u;
}
// act'(u); the ReLU's slope at 0 is 0
template <typename T, int ACT>
__device__ __forceinline__ float act_slope(float u) {
    if (ACT == HGQ_ACT_RELU) return u > 0.f ? 1.f : (u <= 0.f ? 0.f : u);
    if (ACT == HGQ_ACT_SILU) {
        float p, q;
        sigmoid_pair<sizeof(T) == 4>(u, p, q);
        return p + p * (u * q);
    }
    if (ACT == HGQ_ACT_GELU) return 0.5f * (1.f + erff(u * 0.70710678118654752f)) + u * expf(-0.5f * u * u) * 0.39894228040143268f;
    return 1.f;
}

// The body once per activation, the choice outside its loops.
#define GN_FOR_ACT(act, ...)                                             \
    switch (act) {                                                       \
        case HGQ_ACT_RELU: { constexpr int ACT = HGQ_ACT_RELU; __VA_ARGS__; break; } \
        case HGQ_ACT_SILU: { constexpr int ACT = HGQ_ACT_SILU; __VA_ARGS__; break; } \
        case HGQ_ACT_GELU: { constexpr int ACT = HGQ_ACT_GELU; __VA_ARGS__; break; } \
        default: { constexpr int ACT = HGQ_ACT_NONE; __VA_ARGS__; break; }           \
    }

// Packs stay in their own type until they are used, as whole words (16-bit halves in registers of their own would double them).
template <int BYTES> struct Words { using type = uint16_t; };
template <> struct Words<4> { using type = uint32_t; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<16> { using type = uint4; };

__device__ __forceinline__ void unpack_word(uint32_t w, float &lo, float &hi, const __nv_bfloat16 *) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack_word(uint32_t w, float &lo, float &hi, const __half *) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    lo = f.x;
    hi = f.y;
}

template <typename T, int VEC, int R>
struct Held {
    static constexpr int kBytes = (int)sizeof(T) * VEC;
    using W = typename Words<kBytes>::type;
    W q[R];

    __device__ __forceinline__ void load(const T *p, int64_t step, unsigned mask) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            q[j] = W{};
            if (mask >> j & 1) q[j] = *reinterpret_cast<const W *>(p + j * step);
        }
    }
    // The same a sample ahead: 16-byte packs are copied to this thread's places in shared memory while the sample before is worked
    // on (its own packs: no barrier), and taken from there.
    static constexpr bool kAhead = kBytes == 16;
    static constexpr int kStageBytes = kAhead ? R * kThreads * 16 : 0;
    static __device__ __forceinline__ void fetch(unsigned char *stage, const T *p, int64_t step, unsigned mask) {
        uint32_t d = (uint32_t)__cvta_generic_to_shared(stage) + threadIdx.x * 16;
#pragma unroll
        for (int j = 0; j < R; ++j, d += kThreads * 16)
            if (mask >> j & 1) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(p + j * step) : "memory");
    }
    static __device__ __forceinline__ void arrived() { asm volatile("cp.async.wait_all;" ::: "memory"); }
    __device__ __forceinline__ void take(const unsigned char *stage, unsigned mask) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            q[j] = W{};
            if (mask >> j & 1) q[j] = reinterpret_cast<const W *>(stage)[j * kThreads + threadIdx.x];
        }
    }
    __device__ __forceinline__ void values(int j, float (&v)[VEC]) const {
        if constexpr (kBytes == 2) {
            v[0] = to_float(*reinterpret_cast<const T *>(&q[j]));
        } else {
            const uint32_t *w = reinterpret_cast<const uint32_t *>(&q[j]);
#pragma unroll
            for (int k = 0; k < kBytes / 4; ++k) {
                if constexpr (sizeof(T) == 4) v[k] = __uint_as_float(w[k]);
                else unpack_word(w[k], v[2 * k], v[2 * k + 1], (const T *)nullptr);
            }
        }
    }
};

// Samples (or slabs of their channels) that fit on chip: how a call is cut up for the one-read kernels.  usable == false: the
// shape is for the kernels that read twice.
struct SlabPlan {
    bool usable;
    int groups_of_pack;  // numbers that a pack adds to: one a group where packs and groups nest, else one a channel
    int vec;        // channels a thread takes at once
    int q;          // rows taken as one where vec does not divide the channels
    int R;          // packs of one tensor that a thread holds
    int K;          // CTAs of a cluster that share a slab's rows
    int slabs;      // along the channels; Cs channels (whole groups) each, the last one may have fewer
    int Cs, Gs;
    int TX, TY;     // threads along channels and along rows
    int subs;       // samples a CTA works on at once (small ones), TYs thread rows each
    int TYs;
    int rows;       // of one CTA
    int64_t items;  // ceil(B / subs)
    int64_t workers;
    bool ahead;     // forward: the next sample is fetched while this one is worked on
};

SlabPlan gn_slab_plan(int64_t B, int64_t S, int C, int G, int type, int vec, bool backward);
int gn_slab_fwd(const SlabPlan &p, const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, int64_t B,
                int64_t S, int C, int G, float eps, int act, int type, cudaStream_t st);
// part: [workers K][2][C] sums of du and du xhat, written when not NULL
int gn_slab_bwd(const SlabPlan &p, const void *gy, const void *x, const float *gamma, const float *beta, const float *mean,
                const float *rstd, void *dx, float *part, int64_t B, int64_t S, int C, int G, int act, int type, cudaStream_t st);

}  // namespace hgq
