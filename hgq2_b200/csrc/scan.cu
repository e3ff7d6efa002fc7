// Gated linear recurrence over the time axis of [batch, time, features], forward and backward:
//
//   h_t = a_t h_{t-1} + c_t x_t,  a_t = sigmoid(z_t),  c_t = 1 - a_t = sigmoid(-z_t)
//   lambda_t = g_t + a_{t+1} lambda_{t+1};  dx_t = c_t lambda_t;  dz_t = a_t c_t lambda_t (h_{t-1} - x_t);  dh_0 = a_0 lambda_0
//
// A step is the affine map h -> a h + b, and maps compose: (A, H) after (A', H') is (A A', A H' + H).  A lane owns one channel
// (feature of one batch row) for STEPS consecutive time steps held in registers; the warps of a CTA hold consecutive runs of
// the same 32 channels (a tile of WT x STEPS steps).  Each warp folds its run to one map, the maps meet in shared memory, every
// warp folds those before its own onto the tile's incoming state and walks its run again from registers.  x and z are read
// once, all loads of a tile are in flight together, and the state passes from tile to tile in a register: per-channel work in
// time order, so nothing depends on scheduling.  Products of gates stay in (0, 1): there is no division by them and no
// logarithm, so a gate that closes (a = 0) is exact.
//
// Few channels and a long axis leave most SMs without a CTA.  The axis is then cut into segments: a first launch folds each
// segment to one map, the second starts each segment from the fold of the maps before it (x and z are read twice, the second
// time mostly from L2).
//
// The backward pass needs h_{t-1}.  The forward pass keeps the fp32 state at each tile's start (1 / (16 WT) of the outputs) and the
// backward pass recomputes h inside the tile: it never reads h, and gradients of bf16 / fp16 sequences use unrounded states.
//
// Steps at or behind a row's length are the identity map: the state passes through, outputs and gradients there are zero.
// State, maps and gradients are fp32; h, dx, dz are rounded to their type once, on the way out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "hgq_common.cuh"

namespace hgq {

constexpr int kScanSteps = 16;
constexpr int kScanMaxWarps = 16;   // along time
constexpr int kScanMaxSegments = 64;

__device__ __forceinline__ float scan_float(float v) { return v; }
__device__ __forceinline__ float scan_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float scan_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void scan_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void scan_store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void scan_store(__half *p, float v) { *p = __float2half_rn(v); }

struct ScanDims {
    int64_t B, T, D, channels;       // channels = B D
    int64_t xsb, xst, zsb, zst, gsb, gst;  // batch and time strides of x, z and the upstream gradient, in elements
    int64_t dxb, dxt, dzb, dzt;            // and of the gradients of x and z
    int WT, WC;                      // warps of a CTA along time and along channels
    int64_t tiles, tiles_per_segment;
    int segments;
};

// sigmoid(z) and sigmoid(-z), both to full relative precision
__device__ __forceinline__ void gates(float z, float &a, float &c) {
    const float e = expf(-fabsf(z)), r = 1.f / (1.f + e), er = e * r;
    a = z >= 0.f ? r : er;
    c = z >= 0.f ? er : r;
    if (z != z) a = c = z;
}

struct Lane {
    int64_t c, b, d;
    int64_t len;  // steps of this row
    bool in;
    int wt, wc, lane;
};

__device__ __forceinline__ Lane scan_lane(const ScanDims &s, const int32_t *lengths) {
    Lane l;
    const int w = threadIdx.x >> 5;
    l.lane = threadIdx.x & 31;
    l.wt = w % s.WT;
    l.wc = w / s.WT;
    l.c = ((int64_t)blockIdx.x * s.WC + l.wc) * 32 + l.lane;
    l.in = l.c < s.channels;
    l.b = l.in ? l.c / s.D : 0;
    l.d = l.in ? l.c - l.b * s.D : 0;
    l.len = l.in ? s.T : 0;
    if (l.in && lengths != nullptr) {
        const int64_t n = lengths[l.b];
        l.len = n < 0 ? 0 : (n > s.T ? s.T : n);
    }
    return l;
}

// The gates and inputs of STEPS steps from t0; steps that are not live are the identity.
template <typename T, int STEPS>
__device__ __forceinline__ void load_run(const T *__restrict__ x, const T *__restrict__ z, const ScanDims &s, const Lane &l, int64_t t0,
                                         float (&a)[STEPS], float (&c)[STEPS], float (&v)[STEPS]) {
    const T *xp = x + l.b * s.xsb + l.d + t0 * s.xst, *zp = z + l.b * s.zsb + l.d + t0 * s.zst;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const bool live = t0 + i < l.len;
        a[i] = live ? scan_float(zp[i * s.zst]) : 0.f;
        v[i] = live && x != nullptr ? scan_float(xp[i * s.xst]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const float zi = a[i];
        gates(zi, a[i], c[i]);
        if (t0 + i >= l.len) a[i] = 1.f, c[i] = 0.f;
    }
}

// Segment fold, one CTA per (channel tile, segment): agg[segment][channel] = (A, H).
template <typename T, int STEPS>
__global__ void __launch_bounds__(512) k_scan_fold(const T *__restrict__ x, const T *__restrict__ z, const int32_t *__restrict__ lengths,
                                                   const ScanDims s, float2 *__restrict__ agg) {
    __shared__ float2 sh[2][kScanMaxWarps][32];
    const Lane l = scan_lane(s, lengths);
    const int seg = blockIdx.y;
    const int64_t first = seg * s.tiles_per_segment, last = min(s.tiles, first + s.tiles_per_segment);
    float A = 1.f, H = 0.f;
    for (int64_t tile = first; tile < last; ++tile) {
        float a[STEPS], c[STEPS], v[STEPS];
        load_run<T, STEPS>(x, z, s, l, (tile * s.WT + l.wt) * STEPS, a, c, v);
        float ra = 1.f, rh = 0.f;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            rh = a[i] * rh + c[i] * v[i];
            ra *= a[i];
        }
        float2(*buf)[32] = sh[tile & 1];
        buf[l.wc * s.WT + l.wt][l.lane] = make_float2(ra, rh);
        __syncthreads();
        if (l.wt == 0)
            for (int w = 0; w < s.WT; ++w) {
                const float2 q = buf[l.wc * s.WT + w][l.lane];
                H = q.x * H + q.y;
                A *= q.x;
            }
    }
    if (l.wt == 0 && l.in) agg[(int64_t)seg * s.channels + l.c] = make_float2(A, H);
}

template <typename T, int STEPS>
__global__ void __launch_bounds__(512) k_scan_fwd(const T *__restrict__ x, const T *__restrict__ z, const float *__restrict__ h0,
                                                  const int32_t *__restrict__ lengths, const ScanDims s, const float2 *__restrict__ agg,
                                                  T *__restrict__ out, float *__restrict__ h_last, float *__restrict__ states) {
    __shared__ float2 sh[2][kScanMaxWarps][32];
    const Lane l = scan_lane(s, lengths);
    const int seg = blockIdx.y;
    const int64_t first = seg * s.tiles_per_segment, last = min(s.tiles, first + s.tiles_per_segment);
    float carry = (l.in && h0 != nullptr) ? h0[l.c] : 0.f;
    if (l.in)
        for (int k = 0; k < seg; ++k) {
            const float2 q = agg[(int64_t)k * s.channels + l.c];
            carry = q.x * carry + q.y;
        }
    for (int64_t tile = first; tile < last; ++tile) {
        const int64_t t0 = (tile * s.WT + l.wt) * STEPS;
        float a[STEPS], c[STEPS], v[STEPS];
        load_run<T, STEPS>(x, z, s, l, t0, a, c, v);
        if (states != nullptr && l.wt == 0 && l.in) states[tile * s.channels + l.c] = carry;
        float h = carry;
        if (s.WT > 1) {
            float ra = 1.f, rh = 0.f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                v[i] *= c[i];
                rh = a[i] * rh + v[i];
                ra *= a[i];
            }
            float2(*buf)[32] = sh[tile & 1];
            buf[l.wc * s.WT + l.wt][l.lane] = make_float2(ra, rh);
            __syncthreads();
            for (int w = 0; w < s.WT; ++w) {
                if (w == l.wt) h = carry;
                const float2 q = buf[l.wc * s.WT + w][l.lane];
                carry = q.x * carry + q.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) v[i] *= c[i];
        }
        T *op = out + (l.b * s.T + t0) * s.D + l.d;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            h = a[i] * h + v[i];
            if (l.in && t0 + i < s.T) scan_store(op + i * s.D, t0 + i < l.len ? h : 0.f);
        }
        if (s.WT == 1) carry = h;
    }
    if (seg == s.segments - 1 && l.wt == 0 && l.in) h_last[l.c] = carry;
}

// Segment fold of the backward recurrence: agg[segment][channel] = (A, L), the map of the gradient that arrives from the right.
template <typename T, int STEPS>
__global__ void __launch_bounds__(512) k_scan_bwd_fold(const T *__restrict__ gh, const T *__restrict__ z, const int32_t *__restrict__ lengths,
                                                       const ScanDims s, float2 *__restrict__ agg) {
    __shared__ float2 sh[2][kScanMaxWarps][32];
    const Lane l = scan_lane(s, lengths);
    const int seg = blockIdx.y;
    const int64_t first = seg * s.tiles_per_segment, last = min(s.tiles, first + s.tiles_per_segment);
    ScanDims sg = s;
    sg.xsb = s.gsb, sg.xst = s.gst;
    float A = 1.f, L = 0.f;
    for (int64_t tile = last - 1; tile >= first; --tile) {
        float a[STEPS], c[STEPS], g[STEPS];
        load_run<T, STEPS>(gh, z, sg, l, (tile * s.WT + l.wt) * STEPS, a, c, g);
        float ra = 1.f, rl = 0.f;
#pragma unroll
        for (int i = STEPS - 1; i >= 0; --i) {
            rl = a[i] * (g[i] + rl);
            ra *= a[i];
        }
        float2(*buf)[32] = sh[tile & 1];
        buf[l.wc * s.WT + l.wt][l.lane] = make_float2(ra, rl);
        __syncthreads();
        if (l.wt == 0)
            for (int w = s.WT - 1; w >= 0; --w) {
                const float2 q = buf[l.wc * s.WT + w][l.lane];
                L = q.x * L + q.y;
                A *= q.x;
            }
    }
    if (l.wt == 0 && l.in) agg[(int64_t)seg * s.channels + l.c] = make_float2(A, L);
}

template <typename T, int STEPS>
__global__ void __launch_bounds__(512) k_scan_bwd(const T *__restrict__ gh, const T *__restrict__ x, const T *__restrict__ z,
                                                  const float *__restrict__ h0, const int32_t *__restrict__ lengths,
                                                  const float *__restrict__ states, const float *__restrict__ g_last, const ScanDims s,
                                                  const float2 *__restrict__ agg, T *__restrict__ dx, T *__restrict__ dz,
                                                  float *__restrict__ dh0) {
    __shared__ float2 sh[2][kScanMaxWarps][32];
    __shared__ float shl[2][kScanMaxWarps][32];
    const Lane l = scan_lane(s, lengths);
    const int seg = blockIdx.y;
    const int64_t first = seg * s.tiles_per_segment, last = min(s.tiles, first + s.tiles_per_segment);
    float mu = (l.in && g_last != nullptr) ? g_last[l.c] : 0.f;  // gradient of the state behind the tile
    if (l.in)
        for (int k = s.segments - 1; k > seg; --k) {
            const float2 q = agg[(int64_t)k * s.channels + l.c];
            mu = q.x * mu + q.y;
        }
    for (int64_t tile = last - 1; tile >= first; --tile) {
        const int64_t t0 = (tile * s.WT + l.wt) * STEPS;
        float a[STEPS], c[STEPS], v[STEPS], g[STEPS];
        load_run<T, STEPS>(x, z, s, l, t0, a, c, v);
        const T *gp = gh + l.b * s.gsb + l.d + t0 * s.gst;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) g[i] = gh != nullptr && t0 + i < l.len ? scan_float(gp[i * s.gst]) : 0.f;
        float h = 0.f;
        if (l.in) h = states != nullptr ? states[tile * s.channels + l.c] : (h0 != nullptr ? h0[l.c] : 0.f);
        float m = mu;
        if (s.WT > 1) {
            float ra = 1.f, rh = 0.f, rl = 0.f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                rh = a[i] * rh + c[i] * v[i];
                ra *= a[i];
            }
#pragma unroll
            for (int i = STEPS - 1; i >= 0; --i) rl = a[i] * (g[i] + rl);
            const int row = l.wc * s.WT + l.wt, buf = (int)(tile & 1);
            sh[buf][row][l.lane] = make_float2(ra, rh);
            shl[buf][row][l.lane] = rl;
            __syncthreads();
            for (int w = 0; w < l.wt; ++w) {
                const float2 q = sh[buf][l.wc * s.WT + w][l.lane];
                h = q.x * h + q.y;
            }
            for (int w = s.WT - 1; w >= 0; --w) {
                if (w == l.wt) m = mu;
                mu = sh[buf][l.wc * s.WT + w][l.lane].x * mu + shl[buf][l.wc * s.WT + w][l.lane];
            }
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const float d = h - v[i];
            h = a[i] * h + c[i] * v[i];
            v[i] = d;
        }
        T *dxp = dx + l.b * s.dxb + t0 * s.dxt + l.d, *dzp = dz + l.b * s.dzb + t0 * s.dzt + l.d;
#pragma unroll
        for (int i = STEPS - 1; i >= 0; --i) {
            const float lam = g[i] + m;
            const float gx = c[i] * lam;
            m = a[i] * lam;
            if (l.in && t0 + i < s.T) {
                const bool live = t0 + i < l.len;
                scan_store(dxp + i * s.dxt, live ? gx : 0.f);
                scan_store(dzp + i * s.dzt, live ? a[i] * gx * v[i] : 0.f);
            }
        }
        if (s.WT == 1) mu = m;
    }
    if (seg == 0 && l.wt == 0 && l.in && dh0 != nullptr) dh0[l.c] = mu;
}

static int scan_steps(int64_t T) { return T == 1 ? 1 : kScanSteps; }

static ScanDims scan_dims(int64_t B, int64_t T, int64_t D) {
    ScanDims s{};
    s.B = B, s.T = T, s.D = D, s.channels = B * D;
    const int64_t steps = scan_steps(T);
    const int64_t runs = (T + steps - 1) / steps;
    s.WT = 1;
    while (s.WT < runs && s.WT < kScanMaxWarps) s.WT <<= 1;
    s.WC = s.WT < 8 ? 8 / s.WT : 1;
    s.tiles = (runs + s.WT - 1) / s.WT;
    const int64_t ctas = (s.channels + 32 * s.WC - 1) / (32 * s.WC);
    const int64_t sms = num_sms();
    int64_t segments = 1;
    if (ctas < sms && s.tiles > 1) {
        segments = (4 * sms + ctas - 1) / ctas;
        if (segments > kScanMaxSegments) segments = kScanMaxSegments;
        if (segments > s.tiles) segments = s.tiles;
    }
    s.tiles_per_segment = s.tiles > 0 ? (s.tiles + segments - 1) / segments : 0;
    s.segments = s.tiles > 0 ? (int)((s.tiles + s.tiles_per_segment - 1) / s.tiles_per_segment) : 1;
    return s;
}

static int scan_args(int64_t B, int64_t T, int64_t D, int type) {
    if (B < 0 || T < 0 || D < 0) return HGQ_ERR_SIZE;
    if (type < HGQ_TYPE_F32 || type > HGQ_TYPE_F16) return HGQ_ERR_MODE;
    if (D > 0 && B > (int64_t)INT32_MAX * 32 / D) return HGQ_ERR_SIZE;  // grid of 32-channel tiles
    if (B > 0 && D > 0 && T > INT64_MAX / 16 / B / D) return HGQ_ERR_SIZE;
    return HGQ_OK;
}

}  // namespace hgq

using namespace hgq;

extern "C" size_t hgq_gated_scan_workspace(int64_t B, int64_t T, int64_t D) {
    if (scan_args(B, T, D, HGQ_TYPE_F32) != HGQ_OK || B * D == 0) return 0;
    const ScanDims s = scan_dims(B, T, D);
    return s.segments > 1 ? (size_t)s.segments * s.channels * sizeof(float2) : 0;
}

extern "C" int64_t hgq_gated_scan_states(int64_t B, int64_t T, int64_t D) {
    if (scan_args(B, T, D, HGQ_TYPE_F32) != HGQ_OK || B * D == 0) return 0;
    const ScanDims s = scan_dims(B, T, D);
    return s.tiles > 1 ? s.tiles * s.channels : 0;  // one tile starts from h0 itself
}

namespace {

template <typename T>
int scan_fwd(const ScanDims &s, const void *x, const void *z, const float *h0, const int32_t *lengths, void *h, float *h_last, float *states,
             float2 *agg, cudaStream_t st) {
    const dim3 grid((unsigned)((s.channels + 32 * s.WC - 1) / (32 * s.WC)), (unsigned)s.segments);
    const unsigned threads = 32 * s.WT * s.WC;
    if (s.segments > 1) {
        k_scan_fold<T, kScanSteps><<<grid, threads, 0, st>>>((const T *)x, (const T *)z, lengths, s, agg);
        if (int e = check_launch()) return e;
    }
    if (s.T == 1) k_scan_fwd<T, 1><<<grid, threads, 0, st>>>((const T *)x, (const T *)z, h0, lengths, s, agg, (T *)h, h_last, states);
    else k_scan_fwd<T, kScanSteps><<<grid, threads, 0, st>>>((const T *)x, (const T *)z, h0, lengths, s, agg, (T *)h, h_last, states);
    return check_launch();
}

template <typename T>
int scan_bwd(const ScanDims &s, const void *gh, const void *x, const void *z, const float *h0, const int32_t *lengths, const float *states,
             const float *g_last, void *dx, void *dz, float *dh0, float2 *agg, cudaStream_t st) {
    const dim3 grid((unsigned)((s.channels + 32 * s.WC - 1) / (32 * s.WC)), (unsigned)s.segments);
    const unsigned threads = 32 * s.WT * s.WC;
    if (s.segments > 1) {
        k_scan_bwd_fold<T, kScanSteps><<<grid, threads, 0, st>>>((const T *)gh, (const T *)z, lengths, s, agg);
        if (int e = check_launch()) return e;
    }
    if (s.T == 1)
        k_scan_bwd<T, 1><<<grid, threads, 0, st>>>((const T *)gh, (const T *)x, (const T *)z, h0, lengths, states, g_last, s, agg, (T *)dx,
                                                  (T *)dz, dh0);
    else
        k_scan_bwd<T, kScanSteps><<<grid, threads, 0, st>>>((const T *)gh, (const T *)x, (const T *)z, h0, lengths, states, g_last, s, agg,
                                                           (T *)dx, (T *)dz, dh0);
    return check_launch();
}

}  // namespace

extern "C" int hgq_gated_scan_fwd(const void *x, int64_t x_batch, int64_t x_time, const void *z, int64_t z_batch, int64_t z_time,
                                  const float *h0, const int32_t *lengths, void *h, float *h_last, float *states, int64_t B, int64_t T,
                                  int64_t D, int type, void *workspace, size_t workspace_bytes, void *stream) {
    if (int e = scan_args(B, T, D, type)) return e;
    if (B * D == 0) return HGQ_OK;
    if (!h_last || (T > 0 && (!x || !z || !h))) return HGQ_ERR_NULL;
    const size_t size = type == HGQ_TYPE_F32 ? 4 : 2;
    if (!aligned(x, size) || !aligned(z, size) || !aligned(h, size) || !aligned(h0, 4) || !aligned(lengths, 4) || !aligned(h_last, 4) ||
        !aligned(states, 4))
        return HGQ_ERR_ALIGN;
    const size_t need = hgq_gated_scan_workspace(B, T, D);
    if (need > 0 && (!workspace || workspace_bytes < need)) return HGQ_ERR_WORKSPACE;
    if (need > 0 && !aligned(workspace, 8)) return HGQ_ERR_ALIGN;
    ScanDims s = scan_dims(B, T, D);
    s.xsb = x_batch, s.xst = x_time, s.zsb = z_batch, s.zst = z_time;
    if (s.tiles <= 1) states = nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    float2 *agg = (float2 *)workspace;
    if (type == HGQ_TYPE_F32) return scan_fwd<float>(s, x, z, h0, lengths, h, h_last, states, agg, st);
    if (type == HGQ_TYPE_BF16) return scan_fwd<__nv_bfloat16>(s, x, z, h0, lengths, h, h_last, states, agg, st);
    return scan_fwd<__half>(s, x, z, h0, lengths, h, h_last, states, agg, st);
}

extern "C" int hgq_gated_scan_bwd(const void *gh, int64_t g_batch, int64_t g_time, const void *x, int64_t x_batch, int64_t x_time,
                                  const void *z, int64_t z_batch, int64_t z_time, const float *h0, const int32_t *lengths,
                                  const float *states, const float *g_last, void *dx, int64_t dx_batch, int64_t dx_time, void *dz,
                                  int64_t dz_batch, int64_t dz_time, float *dh0, int64_t B, int64_t T, int64_t D, int type, void *workspace, size_t workspace_bytes,
                                  void *stream) {
    if (int e = scan_args(B, T, D, type)) return e;
    if (B * D == 0) return HGQ_OK;
    if (T > 0 && (!x || !z || !dx || !dz)) return HGQ_ERR_NULL;
    const size_t size = type == HGQ_TYPE_F32 ? 4 : 2;
    if (!aligned(gh, size) || !aligned(x, size) || !aligned(z, size) || !aligned(dx, size) || !aligned(dz, size) || !aligned(h0, 4) ||
        !aligned(lengths, 4) || !aligned(states, 4) || !aligned(g_last, 4) || !aligned(dh0, 4))
        return HGQ_ERR_ALIGN;
    const size_t need = hgq_gated_scan_workspace(B, T, D);
    if (need > 0 && (!workspace || workspace_bytes < need)) return HGQ_ERR_WORKSPACE;
    if (need > 0 && !aligned(workspace, 8)) return HGQ_ERR_ALIGN;
    ScanDims s = scan_dims(B, T, D);
    s.xsb = x_batch, s.xst = x_time, s.zsb = z_batch, s.zst = z_time, s.gsb = g_batch, s.gst = g_time;
    s.dxb = dx_batch, s.dxt = dx_time, s.dzb = dz_batch, s.dzt = dz_time;
    if (s.tiles > 1 && !states) return HGQ_ERR_NULL;
    if (s.tiles <= 1) states = nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    float2 *agg = (float2 *)workspace;
    if (type == HGQ_TYPE_F32) return scan_bwd<float>(s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
    if (type == HGQ_TYPE_BF16) return scan_bwd<__nv_bfloat16>(s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
    return scan_bwd<__half>(s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
}
