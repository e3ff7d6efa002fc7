// Gated linear recurrence over the time axis of [batch, time, features], forward and backward:
//
//   h_t = a_t h_{t-1} + c_t x_t,  a_t = sigmoid(z_t),  c_t = 1 - a_t = sigmoid(-z_t)
//   lambda_t = g_t + a_{t+1} lambda_{t+1};  dx_t = c_t lambda_t;  dz_t = a_t c_t lambda_t (h_{t-1} - x_t);  dh_0 = a_0 lambda_0
//
// A step is the affine map h -> a h + b, and maps compose: (A, H) after (A', H') is (A A', A H' + H).  A lane owns VEC neighbouring
// channels (features of one batch row) for kScanSteps consecutive steps held in registers; the WT warps along time of a CTA hold
// consecutive runs of the same channels (a tile).  Each warp folds its run to one map, the maps meet in shared memory, every warp
// folds those before its own onto the tile's incoming state and walks its run again from registers.  x and z are read once, all
// loads of a tile are in flight together, and the state passes from tile to tile in a register: per-channel work in time order,
// so nothing depends on scheduling.  Products of gates stay in [0, 1]: there is no division by them and no logarithm.
//
// Few channels and a long axis leave most SMs without a CTA.  The axis is then cut into segments: a first launch folds each
// segment to one map, the second starts each segment from the fold of the maps before it (x and z are read twice, the second
// time partly from L2: the second launch takes the segments in the opposite order, the last ones read first).
//
// The backward pass needs h_{t-1}.  The forward pass keeps the fp32 state at each tile's start (one number per 64 outputs) and the
// backward pass recomputes h inside the tile: it never reads h, and gradients of bf16 / fp16 sequences use unrounded states.
//
// Steps at or behind a row's length are the identity map: the state passes through, outputs and gradients there are zero.
// State, maps and gradients are fp32; h, dx, dz are rounded to their type once, on the way out.
//
// What bounds it (B200, 6.57 TB/s copy): fp32, memory: [8192, 64, 64] 0.075 ms forward and 0.115 ms backward (0.82 and 0.88 of the copy
// rate for 3 and 5 tensors), [64, 2048, 256] 0.074 and 0.118 ms (0.83, 0.86).  bf16 / fp16: issue slots, 24 to 38 instructions an
// element and pass at half the bytes: [2, 65521, 256] bf16 0.201 ms for both passes in their two launches each.  Padded rows of
// an odd length, [96, 1999, 321] fp16, 0.138 ms forward: issue slots too, 50 instructions an element, half of them for steps behind the
// rows' ends, which are computed like live ones, and accesses of 2 bytes.  What the steps
// gave: expf, IEEE division and a 64-bit multiply per address took 93 instructions an element (0.149 ms for the forward pass of
// [8192, 64, 64]); the gates in fast_sigmoid.cuh, running pointers, two channels a lane and no predicates in full runs 47 (0.070);
// tiles fetched ahead 0.315 -> 0.261 ms for the long bf16 case with a lane's own 4 bytes a copy, 0.201 with 16-byte pieces.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <initializer_list>

#include "fast_sigmoid.cuh"
#include "hgq_common.cuh"

namespace hgq {

constexpr int kScanSteps = 8;
constexpr int kScanMaxWarps = 8;  // along time
constexpr int kScanMaxSegments = 128;
constexpr int kFwdCtas = 3, kBwdCtas = 2;    // CTAs of 256 threads an SM, by their registers, with two channels a lane
constexpr int kFwdCtas1 = 4, kBwdCtas1 = 3;  // and with one

__device__ __forceinline__ float scan_float(float v) { return v; }
__device__ __forceinline__ float scan_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float scan_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void scan_round(float v, float &o) { o = v; }
__device__ __forceinline__ void scan_round(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void scan_round(float v, __half &o) { o = __float2half_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) ScanPack {
    T v[VEC];
};

struct ScanDims {
    int64_t B, T, D, channels;             // channels = B D
    int64_t xsb, xst, zsb, zst, gsb, gst;  // batch and time strides of x, z and the upstream gradient, in elements
    int64_t dxb, dxt, dzb, dzt;            // and of the gradients of x and z
    int WT, WC;                            // warps of a CTA along time and along channels
    int64_t tiles, tiles_per_segment;
    int segments;
};

struct Lane {
    int64_t c, b, d;
    int64_t len;  // steps of this row
    bool in;
    int wt, row, lane;  // row: of this warp in the CTA's exchange buffer, counted from its channel tile's first warp at row - wt
};

// IN_ROWS: lanes do not cross batch rows, for an odd number of features (a kernel's own variant: the arithmetic costs the short
// sequences 0.006 to 0.008 ms of 0.075).  A pair left half empty by the row's end becomes the row's last two channels, one of them its
// neighbour's too (both compute and write the same bits).
template <int VEC, bool IN_ROWS = false>
__device__ __forceinline__ Lane scan_lane(const ScanDims &s, int WT, const int32_t *lengths) {
    Lane l;
    const int w = threadIdx.x >> 5;
    l.lane = threadIdx.x & 31;
    l.wt = w % WT;
    l.row = w;
    if (IN_ROWS) {
        const int64_t p = ((int64_t)blockIdx.x * s.WC + w / WT) * 32 + l.lane, row = (s.D + VEC - 1) / VEC;
        l.in = p < s.B * row;
        l.b = l.in ? p / row : 0;
        l.d = l.in ? (p - l.b * row) * VEC : 0;
        if (l.in && l.d > s.D - VEC) l.d = s.D - VEC;
        l.c = l.b * s.D + l.d;
    } else {
        l.c = (((int64_t)blockIdx.x * s.WC + w / WT) * 32 + l.lane) * VEC;
        l.in = l.c < s.channels;
        l.b = l.in ? l.c / s.D : 0;
        l.d = l.in ? l.c - l.b * s.D : 0;
    }
    l.len = l.in ? s.T : 0;
    if (l.in && lengths != nullptr) {
        const int64_t n = lengths[l.b];
        l.len = n < 0 ? 0 : (n > s.T ? s.T : n);
    }
    return l;
}

// SINGLE: an access for each element, for rows whose packs are not aligned.
template <typename T, int VEC, bool SINGLE>
__device__ __forceinline__ ScanPack<T, VEC> load_pack(const T *__restrict__ p) {
    if (!SINGLE) return *reinterpret_cast<const ScanPack<T, VEC> *>(p);
    ScanPack<T, VEC> q;
#pragma unroll
    for (int k = 0; k < VEC; ++k) q.v[k] = p[k];
    return q;
}

// STEPS packs of a strided sequence as fp32; p: the lane's channel at the first of them, `left`: how many of them are live (the
// others read as zero).
template <typename T, int VEC, int STEPS, bool SINGLE = false>
__device__ __forceinline__ void load_packs(const T *__restrict__ p, int64_t stride, bool full, int64_t left, float (&v)[STEPS][VEC]) {
    using P = ScanPack<T, VEC>;
    P q[STEPS];
    if (full) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i, p += stride) q[i] = load_pack<T, VEC, SINGLE>(p);
    } else {
#pragma unroll
        for (int i = 0; i < STEPS; ++i, p += stride) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) scan_round(0.f, q[i].v[k]);
            if (i < left) q[i] = load_pack<T, VEC, SINGLE>(p);
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[i][k] = scan_float(q[i].v[k]);
}

// The same through shared memory, fetched a tile ahead: a warp's packs of one sequence are STEPS rows of 32 packs, copied as pieces of
// 16 bytes (a quarter to an eighth of the instructions that copies of a lane's own packs take, which cost more issue slots than
// the recurrence).  A piece lies in one batch row; steps that are not live are filled with zeros.  Rows that allow no more: pieces of 8
// bytes still pay for 16-bit types ([64, 2048, 252] bf16 0.071 ms forward against 0.086 with direct loads), not for fp32
// ([64, 2048, 254] 0.127 against 0.096), and pieces of 4 for neither (odd fp32 rows 0.144 against 0.086).  PIECE == 0: not used; < 0: not used, and
// an access for each element of a pack.
template <typename T, int VEC, int STEPS, int N, int PIECE>
struct Stages {
    using P = ScanPack<T, VEC>;
    static constexpr int kPiece = PIECE > 0 ? PIECE : 16;
    static constexpr int kPieces = 32 * (int)sizeof(P) / kPiece;  // of a row
    static constexpr int kRows = 32 / kPieces;                    // rows that one instruction of the warp copies
    static_assert(kRows >= 1, "a row's pieces fit a warp");
    P *base;        // this warp's buffers: [2][N][STEPS][32]
    uint32_t dst;   // where this lane's piece of a buffer's first rows goes
    int row;        // of this lane's piece
    int64_t b, d, len;
    bool in;

    __device__ __forceinline__ Stages(unsigned char *smem, const ScanDims &s, int WT, const int32_t *lengths) {
        const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = lane % kPieces;
        base = reinterpret_cast<P *>(smem) + w * (2 * N * STEPS * 32);
        row = lane / kPieces;
        dst = (uint32_t)__cvta_generic_to_shared(base) + (uint32_t)((row * kPieces + piece) * kPiece);
        const int64_t c = (((int64_t)blockIdx.x * s.WC + w / WT) * 32) * VEC + piece * (kPiece / (int)sizeof(T));
        in = c < s.channels;
        b = in ? c / s.D : 0;
        d = in ? c - b * s.D : 0;
        len = in ? s.T : 0;
        if (in && lengths != nullptr) {
            const int64_t n = lengths[b];
            len = n < 0 ? 0 : (n > s.T ? s.T : n);
        }
    }
    // p: the tensor, NULL for one of zeros
    __device__ __forceinline__ void fetch(int64_t tile, int n, const T *__restrict__ p, int64_t batch, int64_t time, int64_t t0) const {
        const T *src = p + b * batch + d;
        const int64_t left = p != nullptr ? len - t0 : 0;
        uint32_t to = dst + (uint32_t)(((tile & 1) * N + n) * STEPS * 32 * (int)sizeof(P));
#pragma unroll
        for (int i = 0; i < STEPS; i += kRows, to += 32u * kPiece) {
            const bool live = row + i < left;
            const T *q = live ? src + (t0 + row + i) * time : p;
            if (p == nullptr) {
#pragma unroll
                for (int k = 0; k < kPiece; k += 4) asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + k), "r"(0) : "memory");
            } else if (kPiece == 16) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(q), "r"(live ? 16 : 0) : "memory");
            } else {
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(q), "n"(kPiece), "r"(live ? kPiece : 0) : "memory");
            }
        }
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    static __device__ __forceinline__ void wait(bool next_is_on_the_way) {
        if (next_is_on_the_way) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    __device__ __forceinline__ void values(int64_t tile, int n, float (&v)[STEPS][VEC]) const {
        const P *src = base + ((tile & 1) * N + n) * STEPS * 32 + (threadIdx.x & 31);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const P q = src[i * 32];
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[i][k] = scan_float(q.v[k]);
        }
    }
};

template <typename T, int VEC, int STEPS, bool SINGLE = false>
__device__ __forceinline__ void store_packs(T *p, int64_t stride, bool full, int64_t left, const float (&v)[STEPS][VEC]) {
    using P = ScanPack<T, VEC>;
#pragma unroll
    for (int i = 0; i < STEPS; ++i, p += stride) {
        P q;
#pragma unroll
        for (int k = 0; k < VEC; ++k) scan_round(v[i][k], q.v[k]);
        if (full || i < left) {
            if (SINGLE) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) p[k] = q.v[k];
            } else {
                *reinterpret_cast<P *>(p) = q;
            }
        }
    }
}

template <typename T, int VEC, int STEPS>
__device__ __forceinline__ void make_gates(bool full, int64_t left, float (&a)[STEPS][VEC], float (&c)[STEPS][VEC]) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sigmoid_pair<sizeof(T) == 4>(a[i][k], a[i][k], c[i][k]);
    if (!full) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
            if (i >= left) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) a[i][k] = 1.f, c[i][k] = 0.f;
            }
    }
}

template <int VEC>
struct alignas(8 * VEC) Map {  // h -> A h + H for VEC channels
    float A[VEC], H[VEC];
};

// Segment fold of the forward recurrence: agg[segment][channel] = (A, H).
template <typename T, int VEC, int STEPS, int WARPS, int PIECE>
__global__ void __launch_bounds__(256) k_scan_fold(const T *__restrict__ x, const T *__restrict__ z, const int32_t *__restrict__ lengths,
                                                   const ScanDims s, float2 *__restrict__ agg) {
    __shared__ Map<VEC> sh[2][kScanMaxWarps][32];
    const int WT = WARPS > 0 ? WARPS : s.WT;
    const Lane l = scan_lane<VEC>(s, WT, lengths);
    const int seg = blockIdx.y;
    const int64_t first = seg * s.tiles_per_segment, last = min(s.tiles, first + s.tiles_per_segment);
    float A[VEC], H[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) A[k] = 1.f, H[k] = 0.f;
    extern __shared__ __align__(16) unsigned char staging[];
    constexpr bool AHEAD = PIECE > 0;
    const Stages<T, VEC, STEPS, 2, PIECE> stages(staging, s, WT, lengths);
    auto fetch = [&](int64_t tile) {
        const int64_t t0 = (tile * WT + l.wt) * STEPS;
        stages.fetch(tile, 0, z, s.zsb, s.zst, t0);
        stages.fetch(tile, 1, x, s.xsb, s.xst, t0);
        stages.commit();
    };
    if (AHEAD && first < last) fetch(first);
    for (int64_t tile = first; tile < last; ++tile) {
        const int64_t t0 = (tile * WT + l.wt) * STEPS, left = l.len - t0;
        const bool full = __all_sync(0xffffffffu, left >= STEPS);
        float a[STEPS][VEC], c[STEPS][VEC], v[STEPS][VEC];
        if (AHEAD) {
            if (tile + 1 < last) fetch(tile + 1);
            stages.wait(tile + 1 < last);
            stages.values(tile, 0, a);
            stages.values(tile, 1, v);
        } else {
            load_packs<T, VEC, STEPS>(z + l.b * s.zsb + l.d + t0 * s.zst, s.zst, full, left, a);
            load_packs<T, VEC, STEPS>(x + l.b * s.xsb + l.d + t0 * s.xst, s.xst, full, left, v);
        }
        make_gates<T, VEC, STEPS>(full, left, a, c);
        Map<VEC> m;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            float ra = 1.f, rh = 0.f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                rh = a[i][k] * rh + c[i][k] * v[i][k];
                ra *= a[i][k];
            }
            m.A[k] = ra, m.H[k] = rh;
        }
        Map<VEC>(*buf)[32] = sh[tile & 1];
        buf[l.row][l.lane] = m;
        __syncthreads();
        if (l.wt == 0)
#pragma unroll
            for (int w = 0; w < WT; ++w) {
                const Map<VEC> q = buf[l.row + w][l.lane];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    H[k] = q.A[k] * H[k] + q.H[k];
                    A[k] *= q.A[k];
                }
            }
    }
    if (l.wt == 0 && l.in)
#pragma unroll
        for (int k = 0; k < VEC; ++k) agg[(int64_t)seg * s.channels + l.c + k] = make_float2(A[k], H[k]);
}

template <typename T, int VEC, int STEPS, int WARPS, int PIECE>
__global__ void __launch_bounds__(256, VEC == 2 ? kFwdCtas : kFwdCtas1) k_scan_fwd(const T *__restrict__ x, const T *__restrict__ z, const float *__restrict__ h0,
                                                  const int32_t *__restrict__ lengths, const ScanDims s, const float2 *__restrict__ agg,
                                                  T *__restrict__ out, float *__restrict__ h_last, float *__restrict__ states) {
    __shared__ Map<VEC> sh[2][kScanMaxWarps][32];
    const int WT = WARPS > 0 ? WARPS : s.WT;
    const Lane l = scan_lane<VEC>(s, WT, lengths);
    const int seg = s.segments - 1 - blockIdx.y;
    const int64_t first = seg * s.tiles_per_segment, last = min(s.tiles, first + s.tiles_per_segment);
    float carry[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) carry[k] = (l.in && h0 != nullptr) ? h0[l.c + k] : 0.f;
    if (l.in)
#pragma unroll 4
        for (int j = 0; j < seg; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float2 q = agg[(int64_t)j * s.channels + l.c + k];
                carry[k] = q.x * carry[k] + q.y;
            }
    extern __shared__ __align__(16) unsigned char staging[];
    constexpr bool AHEAD = PIECE > 0;
    const Stages<T, VEC, STEPS, 2, PIECE> stages(staging, s, WT, lengths);
    auto fetch = [&](int64_t tile) {
        const int64_t t0 = (tile * WT + l.wt) * STEPS;
        stages.fetch(tile, 0, z, s.zsb, s.zst, t0);
        stages.fetch(tile, 1, x, s.xsb, s.xst, t0);
        stages.commit();
    };
    if (AHEAD && first < last) fetch(first);
    for (int64_t tile = first; tile < last; ++tile) {
        const int64_t t0 = (tile * WT + l.wt) * STEPS, left = l.len - t0;
        const bool full = __all_sync(0xffffffffu, left >= STEPS);
        float a[STEPS][VEC], c[STEPS][VEC], v[STEPS][VEC];
        if (AHEAD) {
            if (tile + 1 < last) fetch(tile + 1);
            stages.wait(tile + 1 < last);
            stages.values(tile, 0, a);
            stages.values(tile, 1, v);
        } else {
            load_packs<T, VEC, STEPS>(z + l.b * s.zsb + l.d + t0 * s.zst, s.zst, full, left, a);
            load_packs<T, VEC, STEPS>(x + l.b * s.xsb + l.d + t0 * s.xst, s.xst, full, left, v);
        }
        make_gates<T, VEC, STEPS>(full, left, a, c);
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[i][k] *= c[i][k];
        if (states != nullptr && l.wt == 0 && l.in)
#pragma unroll
            for (int k = 0; k < VEC; ++k) states[tile * s.channels + l.c + k] = carry[k];
        float h[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[k] = carry[k];
        if (WT > 1) {
            Map<VEC> m;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                float ra = 1.f, rh = 0.f;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    rh = a[i][k] * rh + v[i][k];
                    ra *= a[i][k];
                }
                m.A[k] = ra, m.H[k] = rh;
            }
            Map<VEC>(*buf)[32] = sh[tile & 1];
            buf[l.row][l.lane] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WT; ++w) {
                const Map<VEC> q = buf[l.row - l.wt + w][l.lane];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    if (w == l.wt) h[k] = carry[k];
                    carry[k] = q.A[k] * carry[k] + q.H[k];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                h[k] = a[i][k] * h[k] + v[i][k];
                v[i][k] = h[k];
            }
        if (!full)
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[i][k] = i < left ? v[i][k] : 0.f;
        if (WT == 1)
#pragma unroll
            for (int k = 0; k < VEC; ++k) carry[k] = h[k];
        store_packs<T, VEC, STEPS>(out + (l.b * s.T + t0) * s.D + l.d, s.D, full, l.in ? s.T - t0 : 0, v);
    }
    if (seg == s.segments - 1 && l.wt == 0 && l.in)
#pragma unroll
        for (int k = 0; k < VEC; ++k) h_last[l.c + k] = carry[k];
}

// Segment fold of the backward recurrence: agg[segment][channel] = (A, L), the map of the gradient that arrives from the right.
template <typename T, int VEC, int STEPS, int WARPS, int PIECE>
__global__ void __launch_bounds__(256) k_scan_bwd_fold(const T *__restrict__ gh, const T *__restrict__ z, const int32_t *__restrict__ lengths,
                                                       const ScanDims s, float2 *__restrict__ agg) {
    __shared__ Map<VEC> sh[2][kScanMaxWarps][32];
    const int WT = WARPS > 0 ? WARPS : s.WT;
    const Lane l = scan_lane<VEC, (PIECE < 0)>(s, WT, lengths);
    const int seg = blockIdx.y;
    const int64_t first = seg * s.tiles_per_segment, last = min(s.tiles, first + s.tiles_per_segment);
    float A[VEC], L[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) A[k] = 1.f, L[k] = 0.f;
    extern __shared__ __align__(16) unsigned char staging[];
    constexpr bool AHEAD = PIECE > 0;
    const Stages<T, VEC, STEPS, 2, PIECE> stages(staging, s, WT, lengths);
    auto fetch = [&](int64_t tile) {
        const int64_t t0 = (tile * WT + l.wt) * STEPS;
        stages.fetch(tile, 0, z, s.zsb, s.zst, t0);
        stages.fetch(tile, 1, gh, s.gsb, s.gst, t0);
        stages.commit();
    };
    if (AHEAD && first < last) fetch(last - 1);
    for (int64_t tile = last - 1; tile >= first; --tile) {
        const int64_t t0 = (tile * WT + l.wt) * STEPS, left = l.len - t0;
        const bool full = __all_sync(0xffffffffu, left >= STEPS);
        float a[STEPS][VEC], c[STEPS][VEC], g[STEPS][VEC];
        if (AHEAD) {
            if (tile > first) fetch(tile - 1);
            stages.wait(tile > first);
            stages.values(tile, 0, a);
            stages.values(tile, 1, g);
        } else {
            load_packs<T, VEC, STEPS, (PIECE < 0)>(z + l.b * s.zsb + l.d + t0 * s.zst, s.zst, full, left, a);
            load_packs<T, VEC, STEPS, (PIECE < 0)>(gh + l.b * s.gsb + l.d + t0 * s.gst, s.gst, full && gh != nullptr, gh != nullptr ? left : 0, g);
        }
        make_gates<T, VEC, STEPS>(full, left, a, c);
        Map<VEC> m;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            float ra = 1.f, rl = 0.f;
#pragma unroll
            for (int i = STEPS - 1; i >= 0; --i) {
                rl = a[i][k] * (g[i][k] + rl);
                ra *= a[i][k];
            }
            m.A[k] = ra, m.H[k] = rl;
        }
        Map<VEC>(*buf)[32] = sh[tile & 1];
        buf[l.row][l.lane] = m;
        __syncthreads();
        if (l.wt == 0)
#pragma unroll
            for (int w = WT - 1; w >= 0; --w) {
                const Map<VEC> q = buf[l.row + w][l.lane];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    L[k] = q.A[k] * L[k] + q.H[k];
                    A[k] *= q.A[k];
                }
            }
    }
    if (l.wt == 0 && l.in)
#pragma unroll
        for (int k = 0; k < VEC; ++k) agg[(int64_t)seg * s.channels + l.c + k] = make_float2(A[k], L[k]);
}

template <typename T, int VEC, int STEPS, int WARPS, int PIECE>
__global__ void __launch_bounds__(256, VEC == 2 ? kBwdCtas : kBwdCtas1) k_scan_bwd(const T *__restrict__ gh, const T *__restrict__ x, const T *__restrict__ z,
                                                  const float *__restrict__ h0, const int32_t *__restrict__ lengths,
                                                  const float *__restrict__ states, const float *__restrict__ g_last, const ScanDims s,
                                                  const float2 *__restrict__ agg, T *__restrict__ dx, T *__restrict__ dz,
                                                  float *__restrict__ dh0) {
    __shared__ Map<VEC> sh[2][kScanMaxWarps][32];
    __shared__ float shl[2][kScanMaxWarps][VEC][32];
    const int WT = WARPS > 0 ? WARPS : s.WT;
    const Lane l = scan_lane<VEC, (PIECE < 0)>(s, WT, lengths);
    const int seg = blockIdx.y;  // the fold went through the segments in this order too, each from its end
    const int64_t first = seg * s.tiles_per_segment, last = min(s.tiles, first + s.tiles_per_segment);
    float mu[VEC];  // gradient of the state behind the tile
#pragma unroll
    for (int k = 0; k < VEC; ++k) mu[k] = (l.in && g_last != nullptr) ? g_last[l.c + k] : 0.f;
    if (l.in)
#pragma unroll 4
        for (int j = s.segments - 1; j > seg; --j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float2 q = agg[(int64_t)j * s.channels + l.c + k];
                mu[k] = q.x * mu[k] + q.y;
            }
    extern __shared__ __align__(16) unsigned char staging[];
    constexpr bool AHEAD = PIECE > 0;
    const Stages<T, VEC, STEPS, 3, PIECE> stages(staging, s, WT, lengths);
    auto fetch = [&](int64_t tile) {
        const int64_t t0 = (tile * WT + l.wt) * STEPS;
        stages.fetch(tile, 0, z, s.zsb, s.zst, t0);
        stages.fetch(tile, 1, x, s.xsb, s.xst, t0);
        stages.fetch(tile, 2, gh, s.gsb, s.gst, t0);
        stages.commit();
    };
    if (AHEAD && first < last) fetch(last - 1);
    for (int64_t tile = last - 1; tile >= first; --tile) {
        const int64_t t0 = (tile * WT + l.wt) * STEPS, left = l.len - t0;
        const bool full = __all_sync(0xffffffffu, left >= STEPS);
        float a[STEPS][VEC], c[STEPS][VEC], v[STEPS][VEC], g[STEPS][VEC], h[VEC];
        if (AHEAD) {
            if (tile > first) fetch(tile - 1);
            stages.wait(tile > first);
            stages.values(tile, 0, a);
            stages.values(tile, 1, v);
            stages.values(tile, 2, g);
        } else {
            load_packs<T, VEC, STEPS, (PIECE < 0)>(z + l.b * s.zsb + l.d + t0 * s.zst, s.zst, full, left, a);
            load_packs<T, VEC, STEPS, (PIECE < 0)>(x + l.b * s.xsb + l.d + t0 * s.xst, s.xst, full, left, v);
            load_packs<T, VEC, STEPS, (PIECE < 0)>(gh + l.b * s.gsb + l.d + t0 * s.gst, s.gst, full && gh != nullptr, gh != nullptr ? left : 0, g);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            h[k] = 0.f;
            if (l.in) h[k] = states != nullptr ? states[tile * s.channels + l.c + k] : (h0 != nullptr ? h0[l.c + k] : 0.f);
        }
        make_gates<T, VEC, STEPS>(full, left, a, c);
        float m[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) m[k] = mu[k];
        if (WT > 1) {
            Map<VEC> run;
            const int buf = (int)(tile & 1), base = l.row - l.wt;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                float ra = 1.f, rh = 0.f, rl = 0.f;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    rh = a[i][k] * rh + c[i][k] * v[i][k];
                    ra *= a[i][k];
                }
#pragma unroll
                for (int i = STEPS - 1; i >= 0; --i) rl = a[i][k] * (g[i][k] + rl);
                run.A[k] = ra, run.H[k] = rh;
                shl[buf][l.row][k][l.lane] = rl;
            }
            sh[buf][l.row][l.lane] = run;
            __syncthreads();
            for (int w = 0; w < l.wt; ++w) {
                const Map<VEC> q = sh[buf][base + w][l.lane];
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[k] = q.A[k] * h[k] + q.H[k];
            }
#pragma unroll
            for (int w = WT - 1; w >= 0; --w)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    if (w == l.wt) m[k] = mu[k];
                    mu[k] = sh[buf][base + w][l.lane].A[k] * mu[k] + shl[buf][base + w][k][l.lane];
                }
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float d = h[k] - v[i][k];
                h[k] = a[i][k] * h[k] + c[i][k] * v[i][k];
                v[i][k] = d;
            }
#pragma unroll
        for (int i = STEPS - 1; i >= 0; --i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float lam = g[i][k] + m[k];
                const float gx = c[i][k] * lam;
                m[k] = a[i][k] * lam;
                v[i][k] = a[i][k] * gx * v[i][k];
                g[i][k] = gx;
            }
        if (!full)
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    v[i][k] = i < left ? v[i][k] : 0.f;
                    g[i][k] = i < left ? g[i][k] : 0.f;
                }
        if (WT == 1)
#pragma unroll
            for (int k = 0; k < VEC; ++k) mu[k] = m[k];
        const int64_t rest = l.in ? s.T - t0 : 0;
        store_packs<T, VEC, STEPS, (PIECE < 0)>(dx + l.b * s.dxb + l.d + t0 * s.dxt, s.dxt, full, rest, g);
        store_packs<T, VEC, STEPS, (PIECE < 0)>(dz + l.b * s.dzb + l.d + t0 * s.dzt, s.dzt, full, rest, v);
    }
    if (seg == 0 && l.wt == 0 && l.in && dh0 != nullptr)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dh0[l.c + k] = mu[k];
}

// Tile geometry.  It depends on the shape alone (not on alignment), because the backward pass reads the states that the forward
// pass laid down; VEC only says how many channels a lane takes.
static int scan_steps(int64_t T) { return T == 1 ? 1 : kScanSteps; }

static ScanDims scan_dims(int64_t B, int64_t T, int64_t D, int ctas_per_sm) {
    ScanDims s{};
    s.B = B, s.T = T, s.D = D, s.channels = B * D;
    const int64_t steps = scan_steps(T);
    const int64_t runs = (T + steps - 1) / steps;
    s.WT = 1;
    while (s.WT < runs && s.WT < kScanMaxWarps) s.WT <<= 1;
    s.WC = 8 / s.WT;
    s.tiles = (runs + s.WT - 1) / s.WT;
    // Cut the axis when the channels alone do not give every SM a CTA, into as many segments as run at once: one wave.
    const int64_t ctas = (s.channels + 64 * s.WC - 1) / (64 * s.WC);
    const int64_t sms = num_sms();
    int64_t segments = 1;
    if (ctas < sms && s.tiles > 1) {
        segments = ctas_per_sm * sms / ctas;
        if (segments > kScanMaxSegments) segments = kScanMaxSegments;
        if (segments > s.tiles) segments = s.tiles;
    }
    s.tiles_per_segment = s.tiles > 0 ? (s.tiles + segments - 1) / segments : 0;
    s.segments = s.tiles > 0 ? (int)((s.tiles + s.tiles_per_segment - 1) / s.tiles_per_segment) : 1;
    return s;
}

static unsigned scan_ctas(const ScanDims &s, int vec) {
    const int64_t lanes = s.B * ((s.D + vec - 1) / vec);
    return (unsigned)((lanes + 32 * s.WC - 1) / (32 * s.WC));
}

static int64_t scan_waves(const ScanDims &s, int vec, int per_sm) {
    const int64_t ctas = (int64_t)scan_ctas(s, vec) * s.segments, slots = (int64_t)per_sm * num_sms();
    return (ctas + slots - 1) / slots;
}

// `n` neighbouring channels as one access: a number of features, strides and addresses that keep every pack aligned.
static bool scan_packs(int64_t D, size_t size, int n, std::initializer_list<const void *> ptrs, std::initializer_list<int64_t> strides) {
    if (D % n != 0) return false;
    for (const void *p : ptrs)
        if (!aligned(p, n * size)) return false;
    for (int64_t st : strides)
        if (st % n != 0) return false;
    return true;
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
    int most = 1;
    for (int per_sm : {kFwdCtas, kBwdCtas}) {
        const int n = scan_dims(B, T, D, per_sm).segments;
        most = n > most ? n : most;
    }
    return most > 1 ? (size_t)most * B * D * sizeof(float2) : 0;
}

extern "C" int64_t hgq_gated_scan_states(int64_t B, int64_t T, int64_t D) {
    if (scan_args(B, T, D, HGQ_TYPE_F32) != HGQ_OK || B * D == 0) return 0;
    const ScanDims s = scan_dims(B, T, D, kFwdCtas);
    return s.tiles > 1 ? s.tiles * s.channels : 0;  // one tile starts from h0 itself
}

namespace {

template <typename T, int VEC, int N>
constexpr size_t kStageBytes = (size_t)kScanMaxWarps * 2 * N * kScanSteps * 32 * sizeof(T) * VEC;

template <typename K>
int allow_smem(K kernel, size_t bytes) {
    if (bytes <= (36u << 10)) return HGQ_OK;  // with at most 12 KB of static shared memory beside it
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) cudaGetLastError();
    return (int)e;
}

// What a lane can take of the channels in one access, one or a pair, and the bytes of the pieces that are fetched ahead where a CTA walks
// several tiles (0: direct loads).
//
// Direct loads leave a choice between one channel and a pair a lane, made by the waves of CTAs that the device runs: a wave of pairs
// takes 1.25 (forward) and 13/9 (backward) as long as one of single channels, and holds 1.5 and 1.33 as many channels.  Forward, one
// channel even where pairs are aligned: [64, 2048, 254] fp32 0.086 ms against 0.097, bf16 0.079 against 0.087 (1 wave each),
// [96, 1999, 322] fp16 0.145 against 0.191 (2 each); pairs: [100, 2048, 254] fp32 0.123 against 0.142 (1 and 2), [8192, 256, 46] bf16
// 0.174 against 0.199.  Backward, pairs by single accesses where rows or addresses are odd: [64, 2048, 255] fp32 0.138 against 0.177,
// bf16 0.144 against 0.194 (1 and 2), [96, 1999, 321] fp16 0.284 against 0.303 (2 and 3); one channel: [8192, 256, 47] bf16 0.386 against
// 0.425, [32768, 64, 9] fp32 0.092 against 0.139.
struct ScanAccess {
    int vec, piece;
};

template <typename T, int VEC, int PIECE>
int scan_fwd(const ScanDims &s, const void *x, const void *z, const float *h0, const int32_t *lengths, void *h, float *h_last, float *states,
             float2 *agg, cudaStream_t st) {
    const dim3 grid(scan_ctas(s, VEC), (unsigned)s.segments);
    const unsigned threads = 32 * s.WT * s.WC;
    const T *px = (const T *)x, *pz = (const T *)z;
    T *ph = (T *)h;
    constexpr int W = kScanMaxWarps;
    constexpr size_t bytes = PIECE > 0 ? kStageBytes<T, VEC, 2> : 0;
    if (s.segments > 1) {  // more than one tile: WT is kScanMaxWarps
        auto fold = k_scan_fold<T, VEC, kScanSteps, W, PIECE>;
        if (int e = allow_smem(fold, bytes)) return e;
        fold<<<grid, threads, bytes, st>>>(px, pz, lengths, s, agg);
        if (int e = check_launch()) return e;
    }
    if (s.WT == W) {
        auto fwd = k_scan_fwd<T, VEC, kScanSteps, W, PIECE>;
        if (int e = allow_smem(fwd, bytes)) return e;
        fwd<<<grid, threads, bytes, st>>>(px, pz, h0, lengths, s, agg, ph, h_last, states);
    } else if (s.T == 1) {
        k_scan_fwd<T, VEC, 1, 1, 0><<<grid, threads, 0, st>>>(px, pz, h0, lengths, s, agg, ph, h_last, states);
    } else {
        k_scan_fwd<T, VEC, kScanSteps, 0, 0><<<grid, threads, 0, st>>>(px, pz, h0, lengths, s, agg, ph, h_last, states);
    }
    return check_launch();
}

template <typename T, int VEC, int PIECE>
int scan_bwd(const ScanDims &s, const void *gh, const void *x, const void *z, const float *h0, const int32_t *lengths, const float *states,
             const float *g_last, void *dx, void *dz, float *dh0, float2 *agg, cudaStream_t st) {
    const dim3 grid(scan_ctas(s, VEC), (unsigned)s.segments);
    const unsigned threads = 32 * s.WT * s.WC;
    const T *pg = (const T *)gh, *px = (const T *)x, *pz = (const T *)z;
    T *pdx = (T *)dx, *pdz = (T *)dz;
    constexpr int W = kScanMaxWarps;
    if (s.segments > 1) {
        constexpr size_t bytes = PIECE > 0 ? kStageBytes<T, VEC, 2> : 0;
        auto fold = k_scan_bwd_fold<T, VEC, kScanSteps, W, PIECE>;
        if (int e = allow_smem(fold, bytes)) return e;
        fold<<<grid, threads, bytes, st>>>(pg, pz, lengths, s, agg);
        if (int e = check_launch()) return e;
    }
    if (s.WT == W) {
        constexpr size_t bytes = PIECE > 0 ? kStageBytes<T, VEC, 3> : 0;
        auto bwd = k_scan_bwd<T, VEC, kScanSteps, W, PIECE>;
        if (int e = allow_smem(bwd, bytes)) return e;
        bwd<<<grid, threads, bytes, st>>>(pg, px, pz, h0, lengths, states, g_last, s, agg, pdx, pdz, dh0);
    } else if (s.T == 1) {
        k_scan_bwd<T, VEC, 1, 1, (PIECE < 0 ? PIECE : 0)><<<grid, threads, 0, st>>>(pg, px, pz, h0, lengths, states, g_last, s, agg, pdx, pdz, dh0);
    } else {
        k_scan_bwd<T, VEC, kScanSteps, 0, (PIECE < 0 ? PIECE : 0)><<<grid, threads, 0, st>>>(pg, px, pz, h0, lengths, states, g_last, s, agg, pdx, pdz, dh0);
    }
    return check_launch();
}

ScanAccess scan_access(const ScanDims &s, size_t size, std::initializer_list<const void *> ptrs, std::initializer_list<int64_t> strides) {
    ScanAccess how{scan_packs(s.D, size, 2, ptrs, strides) ? 2 : 1, 0};
    if (s.tiles_per_segment > 1)
        for (int bytes : {16, 8})
            if (how.piece == 0 && (bytes == 16 || size == 2) && scan_packs(s.D, size, bytes / (int)size, ptrs, strides)) how.piece = bytes;
    return how;
}

template <typename T>
int scan_fwd_by(ScanAccess how, const ScanDims &s, const void *x, const void *z, const float *h0, const int32_t *lengths, void *h,
                float *h_last, float *states, float2 *agg, cudaStream_t st) {
    if (how.piece == 16) return scan_fwd<T, 2, 16>(s, x, z, h0, lengths, h, h_last, states, agg, st);
    if (how.piece == 8) return scan_fwd<T, 2, (sizeof(T) == 2 ? 8 : 0)>(s, x, z, h0, lengths, h, h_last, states, agg, st);
    const bool one = s.tiles_per_segment > 1 && 4 * scan_waves(s, 1, kFwdCtas1) <= 5 * scan_waves(s, 2, kFwdCtas);
    if (how.vec == 2 && !one) return scan_fwd<T, 2, 0>(s, x, z, h0, lengths, h, h_last, states, agg, st);
    return scan_fwd<T, 1, 0>(s, x, z, h0, lengths, h, h_last, states, agg, st);
}

template <typename T>
int scan_bwd_by(ScanAccess how, const ScanDims &s, const void *gh, const void *x, const void *z, const float *h0, const int32_t *lengths,
                const float *states, const float *g_last, void *dx, void *dz, float *dh0, float2 *agg, cudaStream_t st) {
    if (how.piece == 16) return scan_bwd<T, 2, 16>(s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
    if (how.piece == 8) return scan_bwd<T, 2, (sizeof(T) == 2 ? 8 : 0)>(s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
    if (how.vec == 1 && s.D > 1 && 13 * scan_waves(s, 2, kBwdCtas) < 9 * scan_waves(s, 1, kBwdCtas1))
        return scan_bwd<T, 2, -1>(s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
    if (how.vec == 2) return scan_bwd<T, 2, 0>(s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
    return scan_bwd<T, 1, 0>(s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
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
    ScanDims s = scan_dims(B, T, D, kFwdCtas);
    s.xsb = x_batch, s.xst = x_time, s.zsb = z_batch, s.zst = z_time;
    if (s.tiles <= 1) states = nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    float2 *agg = (float2 *)workspace;
    const ScanAccess how = scan_access(s, size, {x, z, h}, {x_batch, x_time, z_batch, z_time});
    if (type == HGQ_TYPE_F32) return scan_fwd_by<float>(how, s, x, z, h0, lengths, h, h_last, states, agg, st);
    if (type == HGQ_TYPE_BF16) return scan_fwd_by<__nv_bfloat16>(how, s, x, z, h0, lengths, h, h_last, states, agg, st);
    return scan_fwd_by<__half>(how, s, x, z, h0, lengths, h, h_last, states, agg, st);
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
    ScanDims s = scan_dims(B, T, D, kBwdCtas);
    s.xsb = x_batch, s.xst = x_time, s.zsb = z_batch, s.zst = z_time, s.gsb = g_batch, s.gst = g_time;
    s.dxb = dx_batch, s.dxt = dx_time, s.dzb = dz_batch, s.dzt = dz_time;
    if (s.tiles > 1 && !states) return HGQ_ERR_NULL;
    if (s.tiles <= 1) states = nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    float2 *agg = (float2 *)workspace;
    const std::initializer_list<const void *> ptrs = {gh, x, z, dx, dz};
    const std::initializer_list<int64_t> strides = {g_batch, g_time, x_batch, x_time, z_batch, z_time, dx_batch, dx_time, dz_batch, dz_time};
    const ScanAccess how = scan_access(s, size, ptrs, strides);
    if (type == HGQ_TYPE_F32) return scan_bwd_by<float>(how, s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
    if (type == HGQ_TYPE_BF16) return scan_bwd_by<__nv_bfloat16>(how, s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
    return scan_bwd_by<__half>(how, s, gh, x, z, h0, lengths, states, g_last, dx, dz, dh0, agg, st);
}
