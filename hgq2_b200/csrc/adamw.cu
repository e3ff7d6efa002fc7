// AdamW over a list of tensors in one launch, states in 32 bits or in 8.
//
//   g' = (g grad_scale + l1) c,  c = min(clipnorm / |g grad_scale + l1|_2, 1) over ALL tensors (1 without clipping)
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
// A block is a warp's unit of work (8 elements a lane): per-block maxima are warp reductions and nothing is shared between
// warps.  The (tensor, block) table is built once by the caller; gradient addresses, which change from step to step, travel in
// the kernel's parameters, so a step copies nothing to the device and a captured graph keeps its own.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "hgq_common.cuh"

namespace hgq {

constexpr int kAdamBlock = HGQ_ADAMW_BLOCK;
constexpr int kAdamWarps = 8;
constexpr int kAdamMaxTensors = 512;  // gradient addresses in one launch's parameters (4.6 KB)
constexpr int kNormCtasPerSm = 4;

struct GradTable {
    const void *p[kAdamMaxTensors];
    uint8_t type[kAdamMaxTensors];
};

struct AdamScalars {
    double lr, b1, b2, clipnorm;
    float f_b1, f_1mb1, f_b2, f_1mb2, eps, grad_scale;
};

template <bool VEC>
__device__ __forceinline__ int elem_of(int j, int lane) {
    return VEC ? (j >> 2) * 128 + lane * 4 + (j & 3) : j * 32 + lane;
}

// 8 values of a lane from an array of `type` at p (already at the block's first element); elements >= count read as 0.
template <bool VEC>
__device__ __forceinline__ void load_any(const void *p, int type, int lane, int count, float (&v)[8]) {
    if (VEC) {
        if (type == HGQ_TYPE_F32) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 q = __ldcs(reinterpret_cast<const float4 *>(p) + h * 32 + lane);
                v[4 * h] = q.x, v[4 * h + 1] = q.y, v[4 * h + 2] = q.z, v[4 * h + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint2 q = __ldcs(reinterpret_cast<const uint2 *>(p) + h * 32 + lane);
                const uint32_t u[2] = {q.x, q.y};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float2 f;
                    if (type == HGQ_TYPE_BF16) {
                        f.x = __uint_as_float(u[k] << 16);
                        f.y = __uint_as_float(u[k] & 0xffff0000u);
                    } else {
                        f = __half22float2(*reinterpret_cast<const __half2 *>(&u[k]));
                    }
                    v[4 * h + 2 * k] = f.x;
                    v[4 * h + 2 * k + 1] = f.y;
                }
            }
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
__device__ __forceinline__ void store_any(void *p, int type, int lane, int count, const float (&v)[8]) {
    if (VEC) {
        if (type == HGQ_TYPE_F32) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                __stcs(reinterpret_cast<float4 *>(p) + h * 32 + lane, make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]));
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t u[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (type == HGQ_TYPE_BF16) {
                        const __nv_bfloat162 q = __floats2bfloat162_rn(v[4 * h + 2 * k], v[4 * h + 2 * k + 1]);
                        u[k] = *reinterpret_cast<const uint32_t *>(&q);
                    } else {
                        const __half2 q = __floats2half2_rn(v[4 * h + 2 * k], v[4 * h + 2 * k + 1]);
                        u[k] = *reinterpret_cast<const uint32_t *>(&q);
                    }
                }
                __stcs(reinterpret_cast<uint2 *>(p) + h * 32 + lane, make_uint2(u[0], u[1]));
            }
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

// e4m3 codes: 8 of a lane.  Decoding is exact (every e4m3 value is an fp16 value).
template <bool VEC>
__device__ __forceinline__ void load_codes(const uint8_t *p, int lane, int count, float (&v)[8]) {
    if (VEC) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t q = __ldcs(reinterpret_cast<const uint32_t *>(p) + h * 32 + lane);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q >> (16 * k)), __NV_E4M3);
                const float2 f = __half22float2(__half2(r));
                v[4 * h + 2 * k] = f.x;
                v[4 * h + 2 * k + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = elem_of<false>(j, lane);
            v[j] = 0.f;
            if (e < count) v[j] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)p[e], __NV_E4M3)));
        }
    }
}

// The values are on the e4m3 grid already (or NaN), so the conversion rounds nothing.
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t *p, int lane, int count, const float (&v)[8]) {
    if (VEC) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t q = 0;
#pragma unroll
            for (int k = 0; k < 2; ++k)
                q |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[4 * h + 2 * k], v[4 * h + 2 * k + 1]), __NV_SATFINITE, __NV_E4M3)
                     << (16 * k);
            __stcs(reinterpret_cast<uint32_t *>(p) + h * 32 + lane, q);
        }
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
__device__ __forceinline__ float dithered_e4m3(float u, uint32_t d16) {
    const bool low = u < 0x1p-6f;
    float y = low ? __fadd_rn(u, 0x1p-6f) : u;
    y = __uint_as_float((__float_as_uint(y) + (d16 << 4)) & 0xfff00000u);
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

template <int BITS, bool VEC>
__device__ __forceinline__ void adamw_block(const hgq_adamw_tensor &T, const void *gp, int gtype, int64_t base, int count, int lane,
                                            void *m_, void *v_, float *m_scale, float *v_scale, const AdamScalars &a, float alpha,
                                            float coef, uint32_t step) {
    const int gsize = gtype == HGQ_TYPE_F32 ? 4 : 2;
    const int wsize = T.w_type == HGQ_TYPE_F32 ? 4 : 2;
    const int64_t so = T.offset + base;
    float *const wm = T.master != nullptr ? T.master + base : reinterpret_cast<float *>(T.w) + base;
    float g[8], w[8], m[8], v[8];
    load_any<VEC>(reinterpret_cast<const char *>(gp) + base * gsize, gtype, lane, count, g);
    load_any<VEC>(wm, HGQ_TYPE_F32, lane, count, w);
    if (BITS == 32) {
        load_any<VEC>(reinterpret_cast<float *>(m_) + so, HGQ_TYPE_F32, lane, count, m);
        load_any<VEC>(reinterpret_cast<float *>(v_) + so, HGQ_TYPE_F32, lane, count, v);
    } else {
        load_codes<VEC>(reinterpret_cast<uint8_t *>(m_) + so, lane, count, m);
        load_codes<VEC>(reinterpret_cast<uint8_t *>(v_) + so, lane, count, v);
        const float sm = m_scale[so / kAdamBlock], sv = v_scale[so / kAdamBlock];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m[j] = __fmul_rn(m[j], sm);
            const float r = __fmul_rn(v[j], sv);
            v[j] = __fmul_rn(r, r);
        }
    }
    const float kept = (float)(1.0 - a.lr * T.decay);
    float top_m = 0.f, top_r = 0.f;
    const float l1 = T.l1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float ge = scaled_grad(g[j], a.grad_scale, l1);
        if (a.clipnorm > 0.0) ge = __fmul_rn(ge, coef);
        m[j] = __fadd_rn(__fmul_rn(m[j], a.f_b1), __fmul_rn(ge, a.f_1mb1));
        v[j] = __fadd_rn(__fmul_rn(v[j], a.f_b2), __fmul_rn(__fmul_rn(ge, ge), a.f_1mb2));
        const float root = __fsqrt_rn(v[j]);
        float we = __fsub_rn(__fmul_rn(w[j], kept), __fdiv_rn(__fmul_rn(alpha, m[j]), __fadd_rn(root, a.eps)));
        we = we < T.lo ? T.lo : we;
        we = we > T.hi ? T.hi : we;
        w[j] = we;
        if (BITS == 8) {
            // lanes beyond the tensor's end hold l1-driven values that are not part of the block
            if (!VEC && elem_of<VEC>(j, lane) >= count) m[j] = 0.f, v[j] = 0.f;
            else v[j] = root;
            top_m = fmaxf(top_m, finite_size(m[j]));
            top_r = fmaxf(top_r, finite_size(v[j]));
        }
    }
    store_any<VEC>(wm, HGQ_TYPE_F32, lane, count, w);
    if (T.master != nullptr) store_any<VEC>(reinterpret_cast<char *>(T.w) + base * wsize, T.w_type, lane, count, w);
    if (BITS == 32) {
        store_any<VEC>(reinterpret_cast<float *>(m_) + so, HGQ_TYPE_F32, lane, count, m);
        store_any<VEC>(reinterpret_cast<float *>(v_) + so, HGQ_TYPE_F32, lane, count, v);
        return;
    }
    top_m = fmaxf(warp_max(top_m), 0x1p-100f);
    top_r = fmaxf(warp_max(top_r), 0x1p-100f);
    const float inv_m = __fdiv_rn(256.f, top_m), inv_r = __fdiv_rn(256.f, top_r);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t d = dither_bits((uint32_t)(so + elem_of<VEC>(j, lane)), step);
        const float sm = fabsf(m[j]), sr = v[j];
        const float cm = copysignf(dithered_e4m3(__fmul_rn(sm, inv_m), d & 0xffffu), m[j]);
        float cr = dithered_e4m3(__fmul_rn(sr, inv_r), d >> 16);
        if (sr > 0.f && cr == 0.f) cr = 0x1p-9f;
        // a moment that is not finite is kept as NaN (e4m3 has no infinity)
        m[j] = sm <= 3.402823466e38f ? cm : __int_as_float(0x7fc00000);
        v[j] = sr <= 3.402823466e38f ? cr : __int_as_float(0x7fc00000);
    }
    store_codes<VEC>(reinterpret_cast<uint8_t *>(m_) + so, lane, count, m);
    store_codes<VEC>(reinterpret_cast<uint8_t *>(v_) + so, lane, count, v);
    if (lane == 0) {
        m_scale[so / kAdamBlock] = top_m * (1.f / 256.f);
        v_scale[so / kAdamBlock] = top_r * (1.f / 256.f);
    }
}

__device__ __forceinline__ bool block_is_vector(const hgq_adamw_tensor &T, const void *gp, int gtype, int count) {
    uintptr_t bits = (uintptr_t)T.master;
    if (T.master != nullptr) bits |= (uintptr_t)T.w << 1;  // 8-byte groups of the 16-bit copy
    else bits |= (uintptr_t)T.w;
    bits |= gtype == HGQ_TYPE_F32 ? (uintptr_t)gp : (uintptr_t)gp << 1;
    return count == kAdamBlock && (bits & 15) == 0;
}

// Sum of squares of the scaled gradients, one fp64 partial a CTA (fixed assignment of blocks to warps: the sum does not depend
// on scheduling).
__global__ void __launch_bounds__(kAdamWarps * 32) k_grad_norm(const __grid_constant__ GradTable G, const hgq_adamw_tensor *__restrict__ tensors,
                                                               const int2 *__restrict__ blocks, int64_t n_blocks, int first_tensor,
                                                               float grad_scale, double *__restrict__ part) {
    __shared__ double red[kAdamWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double s = 0.0;
    for (int64_t b = (int64_t)blockIdx.x * kAdamWarps + warp; b < n_blocks; b += (int64_t)gridDim.x * kAdamWarps) {
        const int2 it = __ldg(blocks + b);
        const void *gp = G.p[it.x - first_tensor];
        if (gp == nullptr) continue;
        const int gtype = G.type[it.x - first_tensor];
        const int64_t base = (int64_t)it.y * kAdamBlock, n = tensors[it.x].n;
        const int count = (int)(n - base < kAdamBlock ? n - base : kAdamBlock);
        const float l1 = tensors[it.x].l1;
        const int gsize = gtype == HGQ_TYPE_F32 ? 4 : 2;
        const char *p = reinterpret_cast<const char *>(gp) + base * gsize;
        float g[8];
        const bool vec = count == kAdamBlock && ((uintptr_t)gp & (uintptr_t)(4 * gsize - 1)) == 0;
        if (vec) load_any<true>(p, gtype, lane, count, g);
        else load_any<false>(p, gtype, lane, count, g);
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
__global__ void __launch_bounds__(kAdamWarps * 32) k_adamw(const __grid_constant__ GradTable G, const hgq_adamw_tensor *__restrict__ tensors,
                                                           const int2 *__restrict__ blocks, int64_t n_blocks, int first_tensor,
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
            const double c = a.clipnorm / sqrt(s);
            s_coef = (float)(c > 1.0 ? 1.0 : c);  // a NaN norm stays NaN and reaches every weight
        } else {
            s_coef = 1.f;
        }
    }
    __syncthreads();
    const float alpha = s_alpha, coef = s_coef;
    for (int64_t b = (int64_t)blockIdx.x * kAdamWarps + warp; b < n_blocks; b += (int64_t)gridDim.x * kAdamWarps) {
        const int2 it = __ldg(blocks + b);
        const void *gp = G.p[it.x - first_tensor];
        if (gp == nullptr) continue;  // no gradient this step: the tensor and its states stay as they are
        const int gtype = G.type[it.x - first_tensor];
        const hgq_adamw_tensor T = tensors[it.x];
        const int64_t base = (int64_t)it.y * kAdamBlock;
        const int count = (int)(T.n - base < kAdamBlock ? T.n - base : kAdamBlock);
        if (block_is_vector(T, gp, gtype, count))
            adamw_block<BITS, true>(T, gp, gtype, base, count, lane, m, v, m_scale, v_scale, a, alpha, coef, (uint32_t)t);
        else
            adamw_block<BITS, false>(T, gp, gtype, base, count, lane, m, v, m_scale, v_scale, a, alpha, coef, (uint32_t)t);
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

extern "C" int hgq_adamw_step(const hgq_adamw_tensor *tensors, int64_t n_tensors, const int32_t *blocks, const int64_t *first_block,
                              const void *const *grads, const uint8_t *grad_types, int state_bits, void *m, void *v, float *m_scale,
                              float *v_scale, double lr, double beta1, double beta2, double eps, double grad_scale, double clipnorm,
                              long long *step, unsigned *ticket, void *workspace, size_t workspace_bytes, void *stream) {
    if (n_tensors < 0 || n_tensors > INT32_MAX) return HGQ_ERR_SIZE;
    if (state_bits != 32 && state_bits != 8) return HGQ_ERR_MODE;
    if (!tensors || !blocks || !first_block || !grads || !grad_types || !m || !v || !step || !ticket) return HGQ_ERR_NULL;
    if (state_bits == 8 && (!m_scale || !v_scale)) return HGQ_ERR_NULL;
    if (!aligned(m, 16) || !aligned(v, 16) || !aligned(blocks, 8) || !aligned(tensors, 8) || !aligned(step, 8)) return HGQ_ERR_ALIGN;
    if (n_tensors == 0) return HGQ_OK;
    for (int64_t i = 0; i < n_tensors; ++i) {
        if (first_block[i + 1] < first_block[i]) return HGQ_ERR_SIZE;
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
            const int64_t b0 = first_block[t0], nb = first_block[t0 + cnt] - b0;
            if (nb == 0 && !(pass == 1 && last)) continue;
            const int2 *bt = reinterpret_cast<const int2 *>(blocks) + b0;
            int64_t ctas = (nb + kAdamWarps - 1) / kAdamWarps;
            if (pass == 0) {
                if (ctas > (int64_t)sms * kNormCtasPerSm) ctas = (int64_t)sms * kNormCtasPerSm;
                k_grad_norm<<<(unsigned)ctas, kAdamWarps * 32, 0, st>>>(G, tensors, bt, nb, (int)t0, a.grad_scale, part + n_part);
                n_part += (int)ctas;
            } else {
                if (ctas < 1) ctas = 1;  // nothing to update, but the step is counted
                if (ctas > (int64_t)sms * 8) ctas = (int64_t)sms * 8;
                if (state_bits == 32)
                    k_adamw<32><<<(unsigned)ctas, kAdamWarps * 32, 0, st>>>(G, tensors, bt, nb, (int)t0, m, v, m_scale, v_scale, a, part,
                                                                          n_part, step, ticket, last ? 1 : 0);
                else
                    k_adamw<8><<<(unsigned)ctas, kAdamWarps * 32, 0, st>>>(G, tensors, bt, nb, (int)t0, m, v, m_scale, v_scale, a, part,
                                                                         n_part, step, ticket, last ? 1 : 0);
            }
            if (int e = check_launch()) return e;
        }
    }
    return HGQ_OK;
}
