// AdamW over a list of tensors in one launch, states in 32 bits or in 8.
//
//   g' = (g grad_scale + l1) c,  c = min(clipnorm / |g grad_scale + l1|_2, 1) over ALL tensors (1 without clipping; NaN if the norm is
//        not finite)
//   m  = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2;  alpha = lr sqrt(1 - b2^t) / (1 - b1^t)
//   w  = clamp(w (1 - lr decay) - alpha m / (sqrt(v) + eps), lo, hi)
//
// 8-bit states.  256 consecutive elements of one tensor (a block) share a scale: m and r = sqrt(v) (the root halves the range
// that the code has to span) are stored as e4m3 codes of x * 256 / max|x|.  Both are running means that move by 10 % and 0.1 % a
// step, less than half a step of a 3-bit mantissa, so rounding to nearest would leave most of them where they are for good;
// the rounding is dithered instead: 16 bits of a mix of the element's place and the step number are added below the last kept
// bit, which keeps the mean and is the same on every run.  r is never rounded to zero unless it is zero: it divides the step.
// The update itself uses the fresh 32-bit m and sqrt(v); only what is kept for the next step is rounded.
//
// Every product and sum that leads to a code is written as a single IEEE operation (no contraction), so the codes are a
// function of the inputs alone and not of how the compiler schedules the expression.
//
// A CTA takes 8 neighbouring blocks of a tensor (a chunk) at a time, a block a warp (8 elements a lane): maxima are warp reductions and
// nothing is shared between warps.  The (tensor, chunk) table is built once by the caller; gradient addresses, which change from step
// to step, travel in the kernel's parameters, so a step copies nothing to the device and a captured graph keeps its own.
//
// What bounds it (B200, 6.57 TB/s copy).  32 bits: memory, 28 bytes an element: 30 M elements in 320 tensors 0.124 ms = 6.7 TB/s, with
// the norm's pass over the gradients (0.030 ms) 0.157 ms.  8 bits: latency before anything else.  About 80 instructions an
// element (an IEEE root, two dithered codes and their mix are half of them; 37 go to the half-rate integer pipe) against 14 to 16
// bytes fill 58 % of the issue slots and 45 % of the integer pipe; a warp loads a block, reduces, divides, encodes and stores with
// nothing of its next block on the way, and 80 registers (16 bytes of them spilled) leave 36 % of the warps: the first stall is the
// loads'.  49 M elements with bf16 gradients 0.19 ms = 0.55 of the copy rate, 299 M with clipping 1.24 to 1.29 ms.  Tried and left out, same two cases:
// the next block copied ahead into shared memory (0.20 ms, 1.62 ms: its copies cost more issue slots than the latency they hide),
// prefetches to L2 (0.185, 1.28), four CTAs an SM at 64 registers (0.18, 1.31: spills), neighbouring chunks to one CTA
// instead of every grid-th (0.19, 1.33).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "hgq_common.cuh"

namespace hgq {

constexpr int kAdamBlock = HGQ_ADAMW_BLOCK;
constexpr int kAdamWarps = HGQ_ADAMW_CHUNK / HGQ_ADAMW_BLOCK;
constexpr int kAdamMaxTensors = 512;  // gradient addresses in one launch's parameters (4.6 KB)
constexpr int kNormCtasPerSm = 8;
constexpr int kAdamCtas32 = 3, kAdamCtas8 = 3;  // CTAs an SM, by registers

struct GradTable {
    const void *p[kAdamMaxTensors];
    uint8_t type[kAdamMaxTensors];
};

struct AdamScalars {
    double lr, b1, b2, clipnorm;
    float f_b1, f_1mb1, f_b2, f_1mb2, eps, grad_scale;
};

// Element j of a lane: VEC, 8 neighbours a lane (whole sectors of memory); otherwise every 32nd.
template <bool VEC>
__device__ __forceinline__ int elem_of(int j, int lane) {
    return VEC ? lane * 8 + j : j * 32 + lane;
}

__device__ __forceinline__ void unpack8(const uint4 q, int type, float (&v)[8]) {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (type == HGQ_TYPE_BF16) {
            v[2 * k] = __uint_as_float(u[k] << 16);
            v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[k]));
            v[2 * k] = f.x;
            v[2 * k + 1] = f.y;
        }
    }
}
__device__ __forceinline__ void quad(const float4 q, float *v) { v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w; }

// e4m3 codes: 8 of a lane.  Decoding is exact (every e4m3 value is an fp16 value).
__device__ __forceinline__ void decode8(const uint2 q, float (&v)[8]) {
    const uint32_t u[2] = {q.x, q.y};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u[k >> 1] >> (16 * (k & 1))), __NV_E4M3);
        const float2 f = __half22float2(__half2(r));
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
    }
}
// The values are on the e4m3 grid already (or NaN), so the conversion rounds nothing.
__device__ __forceinline__ uint2 encode8(const float (&v)[8]) {
    uint32_t u[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k)
        u[k >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[2 * k], v[2 * k + 1]), __NV_SATFINITE, __NV_E4M3) << (16 * (k & 1));
    return make_uint2(u[0], u[1]);
}

// 8 values of a lane from an array of `type` at p (already at the block's first element); elements >= count read as 0.  VEC: p is
// aligned to 4 elements, WIDE to 8 fp32.
template <bool VEC>
__device__ __forceinline__ void load_any(const void *p, int type, int lane, int count, bool wide, float (&v)[8]) {
    if (VEC) {
        if (type == HGQ_TYPE_F32) {
            const float *f = reinterpret_cast<const float *>(p) + lane * 8;
            if (wide) {
                asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                             : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                             : "l"(f)
                             : "memory");
            } else {
                quad(reinterpret_cast<const float4 *>(f)[0], v);
                quad(reinterpret_cast<const float4 *>(f)[1], v + 4);
            }
        } else {
            const uint2 *h = reinterpret_cast<const uint2 *>(p) + lane * 2;
            const uint2 a = h[0], b = h[1];
            unpack8(make_uint4(a.x, a.y, b.x, b.y), type, v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = elem_of<false>(j, lane);
            v[j] = 0.f;
            if (e < count) {
                if (type == HGQ_TYPE_F32) v[j] = reinterpret_cast<const float *>(p)[e];
                else if (type == HGQ_TYPE_BF16) v[j] = __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[e]);
                else v[j] = __half2float(reinterpret_cast<const __half *>(p)[e]);
            }
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void store_any(void *p, int type, int lane, int count, bool wide, const float (&v)[8]) {
    if (VEC) {
        if (type == HGQ_TYPE_F32) {
            float *f = reinterpret_cast<float *>(p) + lane * 8;
            if (wide) {
                stcs8(f, v);
            } else {
                reinterpret_cast<float4 *>(f)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4 *>(f)[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else {
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (type == HGQ_TYPE_BF16) {
                    const __nv_bfloat162 q = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
                    u[k] = *reinterpret_cast<const uint32_t *>(&q);
                } else {
                    const __half2 q = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
                    u[k] = *reinterpret_cast<const uint32_t *>(&q);
                }
            }
            uint2 *h = reinterpret_cast<uint2 *>(p) + lane * 2;
            h[0] = make_uint2(u[0], u[1]);
            h[1] = make_uint2(u[2], u[3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = elem_of<false>(j, lane);
            if (e < count) {
                if (type == HGQ_TYPE_F32) reinterpret_cast<float *>(p)[e] = v[j];
                else if (type == HGQ_TYPE_BF16) reinterpret_cast<__nv_bfloat16 *>(p)[e] = __float2bfloat16_rn(v[j]);
                else reinterpret_cast<__half *>(p)[e] = __float2half_rn(v[j]);
            }
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void load_codes(const uint8_t *p, int lane, int count, float (&v)[8]) {
    if (VEC) {
        decode8(reinterpret_cast<const uint2 *>(p)[lane], v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = elem_of<false>(j, lane);
            v[j] = 0.f;
            if (e < count) v[j] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)p[e], __NV_E4M3)));
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t *p, int lane, int count, const float (&v)[8]) {
    if (VEC) {
        __stcs(reinterpret_cast<uint2 *>(p) + lane, encode8(v));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = elem_of<false>(j, lane);
            if (e < count) p[e] = (uint8_t)__nv_cvt_float_to_fp8(v[j], __NV_SATFINITE, __NV_E4M3);
        }
    }
}

// A 32-bit multiply-xorshift mix of an element's place and the step number (odd constants from the fractional parts of the golden
// ratio and of square roots).
__device__ __forceinline__ uint32_t dither_bits(uint32_t place, uint32_t step) {
    uint32_t h = place * 0x9E3779B1u + step * 0x6A09E667u;
    h ^= h >> 16;
    h *= 0xBB67AE85u;
    h ^= h >> 15;
    h *= 0x3C6EF373u;
    return h ^ (h >> 16);
}

// u in [0, 256] to the e4m3 grid (3 mantissa bits above 2^-6, steps of 2^-9 below), up with probability (distance below) / step.
template <bool LOW>  // LOW: u may lie below 2^-6
__device__ __forceinline__ float dithered_e4m3(float u, uint32_t d16) {
    const bool low = LOW && u < 0x1p-6f;
    float y = low ? __fadd_rn(u, 0x1p-6f) : u;
    y = __uint_as_float((__float_as_uint(y) + d16 * 16u) & 0xfff00000u);
    return low ? __fsub_rn(y, 0x1p-6f) : y;
}

__device__ __forceinline__ float finite_size(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;
}

__device__ __forceinline__ float warp_max(float v) {  // of non-negative numbers: their bit patterns order like integers
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

// The scaled gradient as the moments see it, before clipping.
__device__ __forceinline__ float scaled_grad(float g, float grad_scale, float l1) { return __fadd_rn(__fmul_rn(g, grad_scale), l1); }

// The tensor that a CTA is at.  It is the same for all of its threads, and found from the CTA's number alone: branches on it are
// uniform to the compiler too.
struct Current {
    hgq_adamw_tensor t;
    const char *g;
    int gtype, index;
    float kept;     // 1 - lr decay
    bool clamps;    // has a constraint
    bool scales;    // gradient scale, regulariser or clipping
    bool aligned;   // addresses that 4 elements at a time can be read from
    bool wide_g, wide_w;  // 8 fp32 at a time
};

// VEC: the whole block of 256; otherwise element by element.
template <int BITS, bool VEC>
__device__ __forceinline__ void adamw_block(const Current &T, int64_t base, int count, int lane, void *m_, void *v_,
                                            float *m_scale, float *v_scale, const AdamScalars &a, float alpha, float coef, uint32_t step) {
    const int gsize = T.gtype == HGQ_TYPE_F32 ? 4 : 2;
    const int64_t so = T.t.offset + base;
    float *const wm = (T.t.master != nullptr ? T.t.master : reinterpret_cast<float *>(T.t.w)) + base;
    float g[8], w[8], m[8], v[8];
    load_any<VEC>(T.g + base * gsize, T.gtype, lane, count, T.wide_g, g);
    load_any<VEC>(wm, HGQ_TYPE_F32, lane, count, T.wide_w, w);
    if (BITS == 32) {
        load_any<VEC>(reinterpret_cast<float *>(m_) + so, HGQ_TYPE_F32, lane, count, true, m);
        load_any<VEC>(reinterpret_cast<float *>(v_) + so, HGQ_TYPE_F32, lane, count, true, v);
    } else {
        const float sm = m_scale[so / kAdamBlock], sv = v_scale[so / kAdamBlock];
        load_codes<VEC>(reinterpret_cast<uint8_t *>(m_) + so, lane, count, m);
        load_codes<VEC>(reinterpret_cast<uint8_t *>(v_) + so, lane, count, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m[j] = __fmul_rn(m[j], sm);
            const float r = __fmul_rn(v[j], sv);
            v[j] = __fmul_rn(r, r);
        }
    }
    if (T.scales) {
        const float l1 = T.t.l1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[j] = scaled_grad(g[j], a.grad_scale, l1);
            if (a.clipnorm > 0.0) g[j] = __fmul_rn(g[j], coef);
        }
    }
    // of the block: largest and least sizes (NaN passes by), and a sum that is not zero when a moment is not finite
    float top_m = 0.f, top_r = 0.f, least_m = INFINITY, least_r = INFINITY, odd_sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        m[j] = __fadd_rn(__fmul_rn(m[j], a.f_b1), __fmul_rn(g[j], a.f_1mb1));
        v[j] = __fadd_rn(__fmul_rn(v[j], a.f_b2), __fmul_rn(__fmul_rn(g[j], g[j]), a.f_1mb2));
        const float root = __fsqrt_rn(v[j]);
        // the step is a few bits of w: the fast quotient (2 ulp) is far below what is left of it
        w[j] = __fsub_rn(__fmul_rn(w[j], T.kept), __fdividef(__fmul_rn(alpha, m[j]), __fadd_rn(root, a.eps)));
        if (BITS == 8) {
            v[j] = root;
            // lanes beyond the tensor's end hold values driven by the regulariser that are not part of the block
            if (!VEC && elem_of<VEC>(j, lane) >= count) m[j] = v[j] = 0.f;
            top_m = fmaxf(top_m, fabsf(m[j]));
            top_r = fmaxf(top_r, v[j]);
            least_m = fminf(least_m, fabsf(m[j]));
            least_r = fminf(least_r, v[j]);
            odd_sum = fmaf(m[j], 0.f, fmaf(v[j], 0.f, odd_sum));
        }
    }
    if (T.clamps) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // a NaN stays
            w[j] = w[j] < T.t.lo ? T.t.lo : w[j];
            w[j] = w[j] > T.t.hi ? T.t.hi : w[j];
        }
    }
    store_any<VEC>(wm, HGQ_TYPE_F32, lane, count, T.wide_w, w);
    if (T.t.master != nullptr) store_any<VEC>(reinterpret_cast<char *>(T.t.w) + base * (T.t.w_type == HGQ_TYPE_F32 ? 4 : 2), T.t.w_type, lane, count, false, w);
    if (BITS == 32) {
        store_any<VEC>(reinterpret_cast<float *>(m_) + so, HGQ_TYPE_F32, lane, count, true, m);
        store_any<VEC>(reinterpret_cast<float *>(v_) + so, HGQ_TYPE_F32, lane, count, true, v);
        return;
    }
    const bool odd = __any_sync(0xffffffffu, odd_sum != 0.f);
    if (odd) {  // the scale is that of the finite moments; the others are kept as NaN (e4m3 has no infinity)
        top_m = top_r = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            top_m = fmaxf(top_m, finite_size(m[j]));
            top_r = fmaxf(top_r, finite_size(v[j]));
        }
    }
    const float fm = fmaxf(warp_max(top_m), 0x1p-100f), fr = fmaxf(warp_max(top_r), 0x1p-100f);
    const float inv_m = __fdiv_rn(256.f, fm), inv_r = __fdiv_rn(256.f, fr);
    float um[8], ur[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        um[j] = __fmul_rn(fabsf(m[j]), inv_m);
        ur[j] = __fmul_rn(v[j], inv_r);
    }
    const float least = fminf(__fmul_rn(least_m, inv_m), __fmul_rn(least_r, inv_r));
    if (!odd && __all_sync(0xffffffffu, least >= 0x1p-6f)) {  // the usual block: no code below the normal range
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t d = dither_bits((uint32_t)(so + elem_of<VEC>(j, lane)), step);
            m[j] = copysignf(dithered_e4m3<false>(um[j], d & 0xffffu), m[j]);
            v[j] = dithered_e4m3<false>(ur[j], d >> 16);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t d = dither_bits((uint32_t)(so + elem_of<VEC>(j, lane)), step);
            const float cm = copysignf(dithered_e4m3<true>(um[j], d & 0xffffu), m[j]);
            float cr = dithered_e4m3<true>(ur[j], d >> 16);
            if (v[j] > 0.f && cr == 0.f) cr = 0x1p-9f;
            const float nan = __int_as_float(0x7fc00000);
            m[j] = fabsf(m[j]) <= 3.402823466e38f ? cm : nan;
            v[j] = v[j] <= 3.402823466e38f ? cr : nan;
        }
    }
    store_codes<VEC>(reinterpret_cast<uint8_t *>(m_) + so, lane, count, m);
    store_codes<VEC>(reinterpret_cast<uint8_t *>(v_) + so, lane, count, v);
    if (lane == 0) {
        m_scale[so / kAdamBlock] = fm * (1.f / 256.f);
        v_scale[so / kAdamBlock] = fr * (1.f / 256.f);
    }
}

// Sum of squares of the scaled gradients, one fp64 partial a CTA (fixed assignment of blocks to warps: the sum does not depend
// on scheduling).
__global__ void __launch_bounds__(kAdamWarps * 32) k_grad_norm(const __grid_constant__ GradTable G, const hgq_adamw_tensor *__restrict__ tensors,
                                                               const int2 *__restrict__ chunks, int64_t n_chunks, int first_tensor,
                                                               float grad_scale, double *__restrict__ part) {
    __shared__ double red[kAdamWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double s = 0.0;
    for (int64_t c = blockIdx.x; c < n_chunks; c += gridDim.x) {
        const int2 it = chunks[c];
        const void *gp = G.p[it.x - first_tensor];
        if (gp == nullptr) continue;
        const int gtype = G.type[it.x - first_tensor];
        const int64_t base = (int64_t)it.y * HGQ_ADAMW_CHUNK + warp * kAdamBlock, n = tensors[it.x].n;
        if (base >= n) continue;
        const int count = (int)(n - base < kAdamBlock ? n - base : kAdamBlock);
        const float l1 = tensors[it.x].l1;
        const int gsize = gtype == HGQ_TYPE_F32 ? 4 : 2;
        const char *p = reinterpret_cast<const char *>(gp) + base * gsize;
        float g[8];
        const bool vec = count == kAdamBlock && ((uintptr_t)gp & (uintptr_t)(4 * gsize - 1)) == 0;
        if (vec) load_any<true>(p, gtype, lane, count, ((uintptr_t)gp & 31) == 0, g);
        else load_any<false>(p, gtype, lane, count, false, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double ge = (double)scaled_grad(g[j], grad_scale, l1);
            if (vec || elem_of<false>(j, lane) < count) s += ge * ge;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < kAdamWarps; ++w) t += red[w];
        part[blockIdx.x] = t;
    }
}

template <int BITS>
__global__ void __launch_bounds__(kAdamWarps * 32, BITS == 32 ? kAdamCtas32 : kAdamCtas8) k_adamw(const __grid_constant__ GradTable G, const hgq_adamw_tensor *__restrict__ tensors,
                                                           const int2 *__restrict__ chunks, int64_t n_chunks, int first_tensor,
                                                           void *m, void *v, float *m_scale, float *v_scale, const AdamScalars a,
                                                           const double *__restrict__ part, int n_part, long long *step,
                                                           unsigned *ticket, int last_launch) {
    __shared__ float s_alpha, s_coef;
    __shared__ double red[kAdamWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long t = *reinterpret_cast<volatile long long *>(step) + 1;
    if (a.clipnorm > 0.0) {
        double s = 0.0;
        for (int i = threadIdx.x; i < n_part; i += kAdamWarps * 32) s += part[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) red[warp] = s;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        s_alpha = (float)(a.lr * sqrt(1.0 - pow(a.b2, (double)t)) / (1.0 - pow(a.b1, (double)t)));
        if (a.clipnorm > 0.0) {
            double s = 0.0;
            for (int w = 0; w < kAdamWarps; ++w) s += red[w];
            const double norm = sqrt(s), c = a.clipnorm / norm;
            // + 0, or NaN where the norm is infinite or NaN: it reaches every weight (1 / infinity would drop the finite gradients)
            s_coef = (float)((c > 1.0 ? 1.0 : c) + (norm - norm));
        } else {
            s_coef = 1.f;
        }
    }
    __syncthreads();
    const float alpha = s_alpha, coef = s_coef;
    Current T;
    T.index = -1;
    for (int64_t c = blockIdx.x; c < n_chunks; c += gridDim.x) {
        const int2 it = chunks[c];
        if (it.x != T.index) {
            T.index = it.x;
            T.t = tensors[it.x];
            T.g = reinterpret_cast<const char *>(G.p[it.x - first_tensor]);
            T.gtype = G.type[it.x - first_tensor];
            T.kept = (float)(1.0 - a.lr * T.t.decay);
            T.clamps = !(T.t.lo == -INFINITY && T.t.hi == INFINITY);
            T.scales = a.clipnorm > 0.0 || a.grad_scale != 1.f || T.t.l1 != 0.f;
            uintptr_t bits = (uintptr_t)T.t.master;
            bits |= T.t.master != nullptr && T.t.w_type != HGQ_TYPE_F32 ? (uintptr_t)T.t.w << 1 : (uintptr_t)T.t.w;  // 16-bit copy: groups of 8 bytes
            bits |= T.gtype == HGQ_TYPE_F32 ? (uintptr_t)T.g : (uintptr_t)T.g << 1;
            T.aligned = (bits & 15) == 0;
            T.wide_g = ((uintptr_t)T.g & 31) == 0;
            T.wide_w = ((uintptr_t)(T.t.master != nullptr ? (void *)T.t.master : T.t.w) & 31) == 0;
        }
        if (T.g == nullptr) continue;  // no gradient this step: the tensor and its states stay as they are
        const int64_t base = (int64_t)it.y * HGQ_ADAMW_CHUNK + warp * kAdamBlock;
        const int64_t left = T.t.n - base;
        if (left <= 0) continue;
        if (T.aligned && left >= kAdamBlock)
            adamw_block<BITS, true>(T, base, kAdamBlock, lane, m, v, m_scale, v_scale, a, alpha, coef, (uint32_t)t);
        else
            adamw_block<BITS, false>(T, base, (int)(left < kAdamBlock ? left : kAdamBlock), lane, m, v, m_scale, v_scale, a, alpha, coef,
                                     (uint32_t)t);
    }
    if (last_launch && threadIdx.x == 0) {
        // every CTA has read the step number before it takes a ticket; the last one advances it
        if (atomicAdd(ticket, 1u) == gridDim.x - 1) {
            *ticket = 0;
            *step = t;
        }
    }
}

}  // namespace hgq

using namespace hgq;

extern "C" size_t hgq_adamw_workspace(int64_t n_tensors) {
    if (n_tensors <= 0) return 0;
    const int64_t launches = (n_tensors + kAdamMaxTensors - 1) / kAdamMaxTensors;
    return (size_t)launches * num_sms() * kNormCtasPerSm * sizeof(double);
}

extern "C" int hgq_adamw_step(const hgq_adamw_tensor *tensors, int64_t n_tensors, const int32_t *chunks, const int64_t *first_chunk,
                              const void *const *grads, const uint8_t *grad_types, int state_bits, void *m, void *v, float *m_scale,
                              float *v_scale, double lr, double beta1, double beta2, double eps, double grad_scale, double clipnorm,
                              long long *step, unsigned *ticket, void *workspace, size_t workspace_bytes, void *stream) {
    if (n_tensors < 0 || n_tensors > INT32_MAX) return HGQ_ERR_SIZE;
    if (state_bits != 32 && state_bits != 8) return HGQ_ERR_MODE;
    if (!tensors || !chunks || !first_chunk || !grads || !grad_types || !m || !v || !step || !ticket) return HGQ_ERR_NULL;
    if (state_bits == 8 && (!m_scale || !v_scale)) return HGQ_ERR_NULL;
    if (!aligned(m, 32) || !aligned(v, 32) || !aligned(chunks, 8) || !aligned(tensors, 8) || !aligned(step, 8) || !aligned(m_scale, 4) ||
        !aligned(v_scale, 4) || !aligned(ticket, 4))
        return HGQ_ERR_ALIGN;
    if (n_tensors == 0) return HGQ_OK;
    for (int64_t i = 0; i < n_tensors; ++i) {
        if (first_chunk[i + 1] < first_chunk[i]) return HGQ_ERR_SIZE;
        if (grad_types[i] > HGQ_TYPE_F16) return HGQ_ERR_MODE;
        if (grads[i] != nullptr && !aligned(grads[i], grad_types[i] == HGQ_TYPE_F32 ? 4 : 2)) return HGQ_ERR_ALIGN;
    }
    const bool clip = clipnorm > 0.0;
    if (clip && (!workspace || workspace_bytes < hgq_adamw_workspace(n_tensors))) return HGQ_ERR_WORKSPACE;
    if (clip && !aligned(workspace, 8)) return HGQ_ERR_ALIGN;
    cudaStream_t st = (cudaStream_t)stream;
    AdamScalars a;
    a.lr = lr, a.b1 = beta1, a.b2 = beta2, a.clipnorm = clip ? clipnorm : 0.0;
    a.f_b1 = (float)beta1, a.f_1mb1 = (float)(1.0 - beta1), a.f_b2 = (float)beta2, a.f_1mb2 = (float)(1.0 - beta2);
    a.eps = (float)eps, a.grad_scale = (float)grad_scale;
    double *part = (double *)workspace;
    int n_part = 0;
    const int sms = num_sms();
    for (int pass = clip ? 0 : 1; pass < 2; ++pass) {
        for (int64_t t0 = 0; t0 < n_tensors; t0 += kAdamMaxTensors) {
            const int cnt = (int)(n_tensors - t0 < kAdamMaxTensors ? n_tensors - t0 : kAdamMaxTensors);
            const bool last = t0 + cnt == n_tensors;
            GradTable G;
            for (int i = 0; i < cnt; ++i) G.p[i] = grads[t0 + i], G.type[i] = grad_types[t0 + i];
            const int64_t c0 = first_chunk[t0], nc = first_chunk[t0 + cnt] - c0;
            if (nc == 0 && !(pass == 1 && last)) continue;
            const int2 *ct = reinterpret_cast<const int2 *>(chunks) + c0;
            int64_t ctas = nc;
            if (pass == 0) {
                if (ctas > (int64_t)sms * kNormCtasPerSm) ctas = (int64_t)sms * kNormCtasPerSm;
                k_grad_norm<<<(unsigned)ctas, kAdamWarps * 32, 0, st>>>(G, tensors, ct, nc, (int)t0, a.grad_scale, part + n_part);
                n_part += (int)ctas;
            } else {
                if (ctas < 1) ctas = 1;  // nothing to update, but the step is counted
                const int resident = sms * (state_bits == 32 ? kAdamCtas32 : kAdamCtas8);
                if (ctas > resident) ctas = resident;
                auto kernel = state_bits == 32 ? k_adamw<32> : k_adamw<8>;
                kernel<<<(unsigned)ctas, kAdamWarps * 32, 0, st>>>(G, tensors, ct, nc, (int)t0, m, v, m_scale, v_scale, a, part, n_part, step,
                                                                      ticket, last ? 1 : 0);
            }
            if (int e = check_launch()) return e;
        }
    }
    return HGQ_OK;
}
