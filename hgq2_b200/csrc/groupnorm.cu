// Group normalisation with an activation, channels last, forward and backward.
//
//   x [B, S, C] (S: product of the spatial extents), G groups of C / G neighbouring channels, n = S C / G values per (sample, group):
//   xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),  u = xhat gamma + beta,  y = act(u)
//   du = gy act'(u);  dbeta = sum du;  dgamma = sum du xhat;
//   dx = rstd (du gamma - mean(du gamma) - xhat mean(du gamma xhat)),  the means over the (sample, group)
//
// The mean is taken first and the variance from the centred values, so that data whose mean is large against its spread keep
// their variance.  All statistics are fp32 per thread, group totals fp32 or fp64; x, gy, y, dx are fp32, bf16 or fp16 and are
// rounded once, on the way out.  The backward pass recomputes u from x (nothing of y is needed), so a pass moves x and gy in and
// dx out.
//
// This file: the entries, and the kernels for samples that do not fit on chip (the others are in groupnorm_slab.cu).  Those read
// twice: partial statistics per channel of runs of rows, totals in fp64, then the application, in groups of samples small enough
// that the second read finds them in L2.  Bound by latency: a thread loads 4 to 8 packs and then computes with
// nothing on the way, which fills 34 to 42 % of the DRAM rate and 42 to 46 % of the issue slots at 22 to 34 % of the warps (k_gn_stats of
// 16-byte packs of 16-bit types also spills 20 bytes at its 80 registers).  [6, 255, 257, 96] bf16 with SiLU 0.066 ms forward and 0.124 ms
// backward (75 MB a tensor).  One wave of CTAs: two more than the SMs hold
// at once made the backward pass 0.160 ms.
#include "groupnorm.cuh"

namespace hgq {

// ---- any shape: partial statistics, totals, application ---------------------------------------------------------------------
// A CTA takes a run of rows of one sample and a tile of channels; a thread owns VEC neighbouring channels for all of its rows.

// Rows in flight at once, by the registers that a pack and its sums take.
constexpr int kGnRows = 8, kGnApplyRows = 4, kGnBwdRows = 4;
constexpr int kGnFwdCtas = 3, kGnBwdCtas = 2;  // CTAs an SM

struct GnGeom {
    int64_t S, rows_per_chunk;
    int C, G, Cg, TX, TY, tiles, chunks;
};

template <int VEC>
__device__ __forceinline__ bool gn_place(const GnGeom &g, int64_t blk, int &b_rel, int &chunk, int &c0, int &tx, int &ty) {
    const int tile = (int)(blk % g.tiles);
    const int64_t q = blk / g.tiles;
    chunk = (int)(q % g.chunks);
    b_rel = (int)(q / g.chunks);
    tx = threadIdx.x % g.TX;
    ty = threadIdx.x / g.TX;
    c0 = (tile * g.TX + tx) * VEC;
    return ty < g.TY && c0 < g.C;
}

// Which of the rows r, r + TY, ... are before `end`.
template <int ROWS>
__device__ __forceinline__ unsigned rows_left(int64_t r, int64_t end, int TY) {
    const int64_t n = (end - r + TY - 1) / TY;  // r < end
    return n >= ROWS ? (1u << ROWS) - 1 : (1u << (int)n) - 1;
}

// Sum over ty of N values a thread; the result is in the threads of ty == 0.  `sh` has blockDim.x * N floats.
template <int N>
__device__ __forceinline__ void sum_over_ty(float (&v)[N], float *sh, const GnGeom &g, int tx, int ty) {
    const bool in = ty < g.TY;
    for (int i = 0; i < N; ++i)
        if (in) sh[(ty * N + i) * g.TX + tx] = v[i];
    int m = 1;
    while (m < g.TY) m <<= 1;
    for (int o = m >> 1; o > 0; o >>= 1) {
        __syncthreads();
        if (in && ty < o && ty + o < g.TY)
            for (int i = 0; i < N; ++i) sh[(ty * N + i) * g.TX + tx] += sh[((ty + o) * N + i) * g.TX + tx];
    }
    __syncthreads();
    if (in && ty == 0)
        for (int i = 0; i < N; ++i) v[i] = sh[i * g.TX + tx];
}

// Per (sample, chunk, channel): mean and centred sum of squares of its rows.  Sums are taken of x minus the chunk's first row, so
// a large mean costs no digits; if that row is itself the outlier of n rows, the squares lose at most about n 2^-24 of the variance
// (its distance is part of the variance).  The totals' step is in fp64.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, kGnFwdCtas) k_gn_stats(const T *__restrict__ x, const GnGeom g, int64_t b_base, float *__restrict__ part) {
    __shared__ float sh[kThreads * 2 * VEC];
    int b, chunk, c0, tx, ty;
    const bool active = gn_place<VEC>(g, blockIdx.x, b, chunk, c0, tx, ty);
    const int64_t r0 = chunk * g.rows_per_chunk, r1 = min(g.S, r0 + g.rows_per_chunk);
    float acc[2 * VEC], k[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = acc[VEC + i] = k[i] = 0.f;
    const int64_t step = (int64_t)g.TY * g.C;
    if (active) {
        const T *base = x + ((b_base + b) * g.S) * g.C + c0;
        load_pack<T, VEC>(base + r0 * g.C, k);
        for (int64_t r = r0 + ty; r < r1; r += (int64_t)kGnRows * g.TY) {
            Held<T, VEC, kGnRows> h;
            const unsigned mask = rows_left<kGnRows>(r, r1, g.TY);
            h.load(base + r * g.C, step, mask);
#pragma unroll
            for (int j = 0; j < kGnRows; ++j)
                if (mask >> j & 1) {
                    float v[VEC];
                    h.values(j, v);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float d = v[i] - k[i];
                        acc[i] += d;
                        acc[VEC + i] += d * d;
                    }
                }
        }
    }
    sum_over_ty<2 * VEC>(acc, sh, g, tx, ty);
    if (active && ty == 0) {
        const float n = (float)(r1 - r0);
        float *out = part + ((int64_t)b * g.chunks + chunk) * 2 * g.C + c0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float d = acc[i] / n;
            out[i] = k[i] + d;
            out[g.C + i] = fmaxf(acc[VEC + i] - acc[i] * d, 0.f);
        }
    }
}

// Sum over the PER threads of a total (a warp, or the whole block), the same in all of them.
template <int PER>
__device__ __forceinline__ double total_sum(double s, double *sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (PER > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
        __syncthreads();
        s = 0.0;
        for (int w = 0; w < PER / 32; ++w) s += sh[w];
    }
    return s;
}

// PER threads for each (sample, group): the parts' means and squares joined in fp64.
template <int PER>
__global__ void __launch_bounds__(kThreads) k_gn_totals(const float *__restrict__ part, const GnGeom g, int64_t b_base, int64_t pairs, float eps,
                                                        float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ double sh[kThreads / 32];
    const int64_t pair = (int64_t)blockIdx.x * (kThreads / PER) + threadIdx.x / PER;
    const int lane = threadIdx.x % PER;
    if (pair >= pairs) return;
    const int64_t b = pair / g.G;
    const int gr = (int)(pair % g.G);
    const float *base = part + b * g.chunks * 2 * g.C + gr * g.Cg;
    const int items = g.chunks * g.Cg;
    const double total = (double)g.S * g.Cg;
    double s = 0.0;
    for (int i = lane; i < items; i += PER) {
        const int ch = i / g.Cg;
        const int64_t rows = min(g.S - ch * g.rows_per_chunk, g.rows_per_chunk);
        s += (double)rows * base[(int64_t)ch * 2 * g.C + i % g.Cg];
    }
    const double mean = total_sum<PER>(s, sh) / total;
    double q = 0.0;
    for (int i = lane; i < items; i += PER) {
        const int ch = i / g.Cg;
        const int64_t rows = min(g.S - ch * g.rows_per_chunk, g.rows_per_chunk);
        const float *p = base + (int64_t)ch * 2 * g.C + i % g.Cg;
        const double d = p[0] - mean;
        q += p[g.C] + (double)rows * d * d;
    }
    q = total_sum<PER>(q, sh) / total;
    if (lane == 0) {
        mean_out[b_base * g.G + pair] = (float)mean;
        rstd_out[b_base * g.G + pair] = (float)(1.0 / sqrt(q + (double)eps));
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, kGnFwdCtas) k_gn_apply(const T *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta,
                                                       const float *__restrict__ mean, const float *__restrict__ rstd, const GnGeom g,
                                                       int64_t b_base, int act, T *__restrict__ y) {
    int b, chunk, c0, tx, ty;
    if (!gn_place<VEC>(g, blockIdx.x, b, chunk, c0, tx, ty)) return;
    const int64_t r0 = chunk * g.rows_per_chunk, r1 = min(g.S, r0 + g.rows_per_chunk);
    float mu[VEC], sc[VEC], of[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int64_t pair = (b_base + b) * g.G + (c0 + i) / g.Cg;
        mu[i] = mean[pair];
        sc[i] = rstd[pair] * (gamma ? gamma[c0 + i] : 1.f);
        of[i] = beta ? beta[c0 + i] : 0.f;
    }
    const int64_t base = ((b_base + b) * g.S) * g.C + c0, step = (int64_t)g.TY * g.C;
    GN_FOR_ACT(act, {
        for (int64_t r = r0 + ty; r < r1; r += (int64_t)kGnApplyRows * g.TY) {
            Held<T, VEC, kGnApplyRows> h;
            const unsigned mask = rows_left<kGnApplyRows>(r, r1, g.TY);
            h.load(x + base + r * g.C, step, mask);
            _Pragma("unroll") for (int j = 0; j < kGnApplyRows; ++j) if (mask >> j & 1) {
                float v[VEC];
                h.values(j, v);
                _Pragma("unroll") for (int i = 0; i < VEC; ++i) v[i] = act_value<T, ACT>((v[i] - mu[i]) * sc[i] + of[i]);
                store_pack<T, VEC>(y + base + r * g.C + j * step, v);
            }
        }
    })
}

// Per (sample, chunk, channel): sum of du and of du xhat.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, kGnBwdCtas) k_gn_bwd_stats(const T *__restrict__ gy, const T *__restrict__ x, const float *__restrict__ gamma,
                                                           const float *__restrict__ beta, const float *__restrict__ mean,
                                                           const float *__restrict__ rstd, const GnGeom g, int64_t b_base, int act,
                                                           float *__restrict__ part) {
    __shared__ float sh[kThreads * 2 * VEC];
    int b, chunk, c0, tx, ty;
    const bool active = gn_place<VEC>(g, blockIdx.x, b, chunk, c0, tx, ty);
    const int64_t r0 = chunk * g.rows_per_chunk, r1 = min(g.S, r0 + g.rows_per_chunk);
    float acc[2 * VEC];
#pragma unroll
    for (int i = 0; i < 2 * VEC; ++i) acc[i] = 0.f;
    if (active) {
        float mu[VEC], rs[VEC], ga[VEC], be[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int64_t pair = (b_base + b) * g.G + (c0 + i) / g.Cg;
            mu[i] = mean[pair];
            rs[i] = rstd[pair];
            ga[i] = gamma ? gamma[c0 + i] : 1.f;
            be[i] = beta ? beta[c0 + i] : 0.f;
        }
        const int64_t base = ((b_base + b) * g.S) * g.C + c0, step = (int64_t)g.TY * g.C;
        GN_FOR_ACT(act, {
            for (int64_t r = r0 + ty; r < r1; r += (int64_t)kGnBwdRows * g.TY) {
                Held<T, VEC, kGnBwdRows> h, hg;
                const unsigned mask = rows_left<kGnBwdRows>(r, r1, g.TY);
                h.load(x + base + r * g.C, step, mask);
                hg.load(gy + base + r * g.C, step, mask);
                _Pragma("unroll") for (int j = 0; j < kGnBwdRows; ++j) if (mask >> j & 1) {
                    float v[VEC], d[VEC];
                    h.values(j, v);
                    hg.values(j, d);
                    _Pragma("unroll") for (int i = 0; i < VEC; ++i) {
                        const float xh = (v[i] - mu[i]) * rs[i];
                        const float du = d[i] * act_slope<T, ACT>(xh * ga[i] + be[i]);
                        acc[i] += du;
                        acc[VEC + i] += du * xh;
                    }
                }
            }
        })
    }
    sum_over_ty<2 * VEC>(acc, sh, g, tx, ty);
    if (active && ty == 0) {
        float *out = part + ((int64_t)b * g.chunks + chunk) * 2 * g.C + c0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = acc[i], out[g.C + i] = acc[VEC + i];
    }
}

// PER threads for each (sample, group): the two means of the backward formula, in fp64.
template <int PER>
__global__ void __launch_bounds__(kThreads) k_gn_bwd_totals(const float *__restrict__ part, const float *__restrict__ gamma, const GnGeom g,
                                                            int64_t pairs, float *__restrict__ m1, float *__restrict__ m2) {
    __shared__ double sh[kThreads / 32];
    const int64_t pair = (int64_t)blockIdx.x * (kThreads / PER) + threadIdx.x / PER;
    const int lane = threadIdx.x % PER;
    if (pair >= pairs) return;
    const int64_t b = pair / g.G;
    const int gr = (int)(pair % g.G);
    const float *base = part + b * g.chunks * 2 * g.C + gr * g.Cg;
    const int items = g.chunks * g.Cg;
    double s1 = 0.0, s2 = 0.0;
    for (int i = lane; i < items; i += PER) {
        const int ch = i / g.Cg, c = i % g.Cg;
        const double ga = gamma ? gamma[gr * g.Cg + c] : 1.f;
        const float *p = base + (int64_t)ch * 2 * g.C + c;
        s1 += ga * p[0];
        s2 += ga * p[g.C];
    }
    s1 = total_sum<PER>(s1, sh);
    s2 = total_sum<PER>(s2, sh);
    if (lane == 0) {
        const double total = (double)g.S * g.Cg;
        m1[pair] = (float)(s1 / total);
        m2[pair] = (float)(s2 / total);
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, kGnBwdCtas) k_gn_bwd_apply(const T *__restrict__ gy, const T *__restrict__ x, const float *__restrict__ gamma,
                                                           const float *__restrict__ beta, const float *__restrict__ mean,
                                                           const float *__restrict__ rstd, const float *__restrict__ m1,
                                                           const float *__restrict__ m2, const GnGeom g, int64_t b_base, int act,
                                                           T *__restrict__ dx) {
    int b, chunk, c0, tx, ty;
    if (!gn_place<VEC>(g, blockIdx.x, b, chunk, c0, tx, ty)) return;
    const int64_t r0 = chunk * g.rows_per_chunk, r1 = min(g.S, r0 + g.rows_per_chunk);
    float mu[VEC], rs[VEC], ga[VEC], be[VEC], a1[VEC], a2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int64_t rel = (int64_t)b * g.G + (c0 + i) / g.Cg, pair = b_base * g.G + rel;
        mu[i] = mean[pair];
        rs[i] = rstd[pair];
        ga[i] = gamma ? gamma[c0 + i] : 1.f;
        be[i] = beta ? beta[c0 + i] : 0.f;
        a1[i] = m1[rel];
        a2[i] = m2[rel];
    }
    const int64_t base = ((b_base + b) * g.S) * g.C + c0, step = (int64_t)g.TY * g.C;
    GN_FOR_ACT(act, {
        for (int64_t r = r0 + ty; r < r1; r += (int64_t)kGnBwdRows * g.TY) {
            Held<T, VEC, kGnBwdRows> h, hg;
            const unsigned mask = rows_left<kGnBwdRows>(r, r1, g.TY);
            h.load(x + base + r * g.C, step, mask);
            hg.load(gy + base + r * g.C, step, mask);
            _Pragma("unroll") for (int j = 0; j < kGnBwdRows; ++j) if (mask >> j & 1) {
                float v[VEC], d[VEC];
                h.values(j, v);
                hg.values(j, d);
                _Pragma("unroll") for (int i = 0; i < VEC; ++i) {
                    const float xh = (v[i] - mu[i]) * rs[i];
                    const float du = d[i] * act_slope<T, ACT>(xh * ga[i] + be[i]);
                    v[i] = rs[i] * (du * ga[i] - a1[i] - xh * a2[i]);
                }
                store_pack<T, VEC>(dx + base + r * g.C + j * step, v);
            }
        }
    })
}

// Column sums of [rows, C2] in a fixed order: 32 columns x 8 row lanes a CTA, grid.y row blocks (a second launch with one block
// sums the blocks' results).
__global__ void __launch_bounds__(kThreads) k_gn_colsum(const float *__restrict__ part, int64_t rows, int64_t C2, float *__restrict__ out,
                                                        float *__restrict__ out2) {
    __shared__ double sh[8][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int ry = threadIdx.x >> 5;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
    double s = 0.0;
    if (c < C2)
        for (int64_t r = r0 + ry; r < r1; r += 8) s += part[r * C2 + c];
    sh[ry][threadIdx.x & 31] = s;
    __syncthreads();
    if (ry == 0 && c < C2) {
        for (int i = 1; i < 8; ++i) s += sh[i][threadIdx.x];
        if (out2 == nullptr) out[blockIdx.y * C2 + c] = (float)s;
        else if (c < C2 / 2) out[c] = (float)s;  // last stage: dbeta first, then dgamma
        else out2[c - C2 / 2] = (float)s;
    }
}

// Samples whose x (and gy) an L2 of 126 MB still holds when the second pass comes back to them.
constexpr int64_t kGnGroupBytes = 80ll << 20;
constexpr int kGnSumBlocks = 64;

static int64_t gn_group(int64_t B, int64_t S, int C, int64_t bytes_per_value) {
    const int64_t sample = S * C * bytes_per_value;
    int64_t n = sample > 0 ? kGnGroupBytes / sample : B;
    if (n < 1) n = 1;
    // equal groups
    const int64_t groups = (B + n - 1) / n;
    return groups > 0 ? (B + groups - 1) / groups : 1;
}

// ctas_per_sm: how many of the call's CTAs an SM holds (their registers): one wave of them, so that no few stragglers follow it.
static GnGeom gn_geom(int64_t group, int64_t S, int C, int G, int vec, int ctas_per_sm) {
    GnGeom g;
    g.S = S, g.C = C, g.G = G, g.Cg = C / G;
    const int cv = C / vec;
    g.tiles = (cv + kThreads - 1) / kThreads;
    g.TX = (cv + g.tiles - 1) / g.tiles;
    g.TY = kThreads / g.TX;
    int64_t chunks = (int64_t)num_sms() * ctas_per_sm / (group * g.tiles);
    const int64_t most = (S + (int64_t)g.TY * 4 - 1) / ((int64_t)g.TY * 4);
    if (chunks > most) chunks = most;
    if (chunks < 1) chunks = 1;
    g.rows_per_chunk = (S + chunks - 1) / chunks;
    g.chunks = (int)((S + g.rows_per_chunk - 1) / g.rows_per_chunk);
    return g;
}

// The widest pack that the addresses and the channel count allow.
static int gn_vec(const void *a, const void *b, const void *c, int C, int type) {
    const int size = type == HGQ_TYPE_F32 ? 4 : 2;
    for (int v : {16 / size, 4, 2})
        if (C % v == 0 && aligned(a, (size_t)v * size) && aligned(b, (size_t)v * size) && aligned(c, (size_t)v * size)) return v;
    return 1;
}

// The one-read plan with the widest pack that the addresses allow (usable == false: none); rows may be joined to make packs fit.
static SlabPlan gn_plan(const void *a, const void *b, const void *c, int64_t B, int64_t S, int C, int G, int type, bool bwd) {
    const int size = type == HGQ_TYPE_F32 ? 4 : 2;
    SlabPlan p{};
    for (int v : {16 / size, 4, 2, 1}) {
        if (!aligned(a, (size_t)v * size) || !aligned(b, (size_t)v * size) || !aligned(c, (size_t)v * size)) continue;
        p = gn_slab_plan(B, S, C, G, type, v, bwd);
        if (p.usable) return p;
    }
    return p;
}

// Partial sums of a call, for whichever access width its addresses allow (the one-read forward pass has none).
static size_t gn_part_floats(int64_t B, int64_t S, int C, int G, int type, bool bwd) {
    const int size = type == HGQ_TYPE_F32 ? 4 : 2;
    const int64_t group = gn_group(B, S, C, bwd ? 2 * size : size);
    size_t most = 0;
    for (int v : {16 / size, 4, 2, 1}) {
        const SlabPlan p = gn_slab_plan(B, S, C, G, type, v, bwd);
        size_t n = p.usable && bwd ? (size_t)p.workers * p.K * 2 * C : 0;
        most = n > most ? n : most;
        if (C % v != 0) continue;
        const GnGeom g = gn_geom(group, S, C, G, v, bwd ? kGnBwdCtas : kGnFwdCtas);
        n = p.usable ? 0 : (size_t)g.chunks * 2 * C * (size_t)(bwd ? B : group);
        most = n > most ? n : most;
    }
    return most;
}

static bool gn_args_ok(int64_t B, int64_t S, int C, int G, int act, int type, int *err) {
    *err = HGQ_OK;
    if (B < 0 || S < 0 || C <= 0 || G <= 0 || C % G != 0) *err = HGQ_ERR_SIZE;
    else if (act < HGQ_ACT_NONE || act > HGQ_ACT_GELU || type < HGQ_TYPE_F32 || type > HGQ_TYPE_F16) *err = HGQ_ERR_MODE;
    else if (B > INT32_MAX || (S > 0 && B > 0 && (S > INT64_MAX / 16 / C || B > INT64_MAX / 16 / C / S))) *err = HGQ_ERR_SIZE;
    return *err == HGQ_OK;
}

template <typename T, int VEC>
static int gn_fwd_any(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, int64_t B, int64_t S, int C,
                      int G, float eps, int act, float *part, cudaStream_t st) {
    const int64_t group = gn_group(B, S, C, sizeof(T));
    const GnGeom g = gn_geom(group, S, C, G, VEC, kGnFwdCtas);
    for (int64_t b0 = 0; b0 < B; b0 += group) {
        const int64_t nb = B - b0 < group ? B - b0 : group, pairs = nb * G;
        const int64_t ctas = nb * g.chunks * g.tiles;
        // parts of a total: a block for each where they are many or the totals few, else a warp
        const bool wide = (int64_t)g.chunks * g.Cg > 256 || ((int64_t)g.chunks * g.Cg > 32 && pairs < 16 * num_sms());
        const int64_t sums = wide ? pairs : (pairs + kThreads / 32 - 1) / (kThreads / 32);
        if (ctas > INT32_MAX || sums > INT32_MAX || (int64_t)g.chunks * g.Cg > INT32_MAX) return HGQ_ERR_SIZE;
        k_gn_stats<T, VEC><<<(unsigned)ctas, kThreads, 0, st>>>((const T *)x, g, b0, part);
        if (int e = check_launch()) return e;
        if (wide) k_gn_totals<kThreads><<<(unsigned)sums, kThreads, 0, st>>>(part, g, b0, pairs, eps, mean, rstd);
        else k_gn_totals<32><<<(unsigned)sums, kThreads, 0, st>>>(part, g, b0, pairs, eps, mean, rstd);
        if (int e = check_launch()) return e;
        k_gn_apply<T, VEC><<<(unsigned)ctas, kThreads, 0, st>>>((const T *)x, gamma, beta, mean, rstd, g, b0, act, (T *)y);
        if (int e = check_launch()) return e;
    }
    return HGQ_OK;
}

static int gn_colsum(const float *part, int64_t rows, int C, float *scratch, float *dgamma, float *dbeta, cudaStream_t st) {
    const unsigned cb = (unsigned)((2 * (int64_t)C + 31) / 32);
    const int64_t rb = rows > 256 ? kGnSumBlocks : 1;
    const float *src = part;
    if (rb > 1) {
        k_gn_colsum<<<dim3(cb, (unsigned)rb), kThreads, 0, st>>>(part, rows, 2 * (int64_t)C, scratch, nullptr);
        if (int e = check_launch()) return e;
        src = scratch;
        rows = rb;
    }
    k_gn_colsum<<<dim3(cb, 1), kThreads, 0, st>>>(src, rows, 2 * (int64_t)C, dbeta, dgamma);
    return check_launch();
}

template <typename T, int VEC>
static int gn_bwd_any(const void *gy, const void *x, const float *gamma, const float *beta, const float *mean, const float *rstd, void *dx,
                      float *dgamma, float *dbeta, int64_t B, int64_t S, int C, int G, int act, float *part, float *m, float *scratch,
                      cudaStream_t st) {
    const int64_t group = gn_group(B, S, C, 2 * sizeof(T));
    const GnGeom g = gn_geom(group, S, C, G, VEC, kGnBwdCtas);
    for (int64_t b0 = 0; b0 < B; b0 += group) {
        const int64_t nb = B - b0 < group ? B - b0 : group, pairs = nb * G;
        const int64_t ctas = nb * g.chunks * g.tiles;
        // parts of a total: a block for each where they are many or the totals few, else a warp
        const bool wide = (int64_t)g.chunks * g.Cg > 256 || ((int64_t)g.chunks * g.Cg > 32 && pairs < 16 * num_sms());
        const int64_t sums = wide ? pairs : (pairs + kThreads / 32 - 1) / (kThreads / 32);
        if (ctas > INT32_MAX || sums > INT32_MAX || (int64_t)g.chunks * g.Cg > INT32_MAX) return HGQ_ERR_SIZE;
        float *p = part + b0 * g.chunks * 2 * C;
        k_gn_bwd_stats<T, VEC><<<(unsigned)ctas, kThreads, 0, st>>>((const T *)gy, (const T *)x, gamma, beta, mean, rstd, g, b0, act, p);
        if (int e = check_launch()) return e;
        if (dx != nullptr) {
            if (wide) k_gn_bwd_totals<kThreads><<<(unsigned)sums, kThreads, 0, st>>>(p, gamma, g, pairs, m, m + group * G);
            else k_gn_bwd_totals<32><<<(unsigned)sums, kThreads, 0, st>>>(p, gamma, g, pairs, m, m + group * G);
            if (int e = check_launch()) return e;
            k_gn_bwd_apply<T, VEC><<<(unsigned)ctas, kThreads, 0, st>>>((const T *)gy, (const T *)x, gamma, beta, mean, rstd, m, m + group * G, g,
                                                                       b0, act, (T *)dx);
            if (int e = check_launch()) return e;
        }
    }
    if (dgamma == nullptr) return HGQ_OK;
    return gn_colsum(part, B * g.chunks, C, scratch, dgamma, dbeta, st);
}

}  // namespace hgq

using namespace hgq;

extern "C" size_t hgq_group_norm_workspace(int64_t B, int64_t S, int C, int G, int type, int backward) {
    int e;
    if (!gn_args_ok(B, S, C, G, HGQ_ACT_NONE, type, &e) || B == 0 || S == 0) return 0;
    const int size = type == HGQ_TYPE_F32 ? 4 : 2;
    size_t n = gn_part_floats(B, S, C, G, type, backward != 0);
    if (backward) n += 2 * (size_t)gn_group(B, S, C, 2 * size) * G + (size_t)kGnSumBlocks * 2 * C;
    return n * sizeof(float);
}

#define GN_DISPATCH(FN, ...)                                                                          \
    do {                                                                                              \
        if (type == HGQ_TYPE_F32) {                                                                   \
            if (vec == 4) return FN<float, 4>(__VA_ARGS__);                                           \
            if (vec == 2) return FN<float, 2>(__VA_ARGS__);                                           \
            return FN<float, 1>(__VA_ARGS__);                                                         \
        }                                                                                             \
        if (type == HGQ_TYPE_BF16) {                                                                  \
            if (vec == 8) return FN<__nv_bfloat16, 8>(__VA_ARGS__);                                   \
            if (vec == 4) return FN<__nv_bfloat16, 4>(__VA_ARGS__);                                   \
            if (vec == 2) return FN<__nv_bfloat16, 2>(__VA_ARGS__);                                   \
            return FN<__nv_bfloat16, 1>(__VA_ARGS__);                                                 \
        }                                                                                             \
        if (vec == 8) return FN<__half, 8>(__VA_ARGS__);                                              \
        if (vec == 4) return FN<__half, 4>(__VA_ARGS__);                                              \
        if (vec == 2) return FN<__half, 2>(__VA_ARGS__);                                              \
        return FN<__half, 1>(__VA_ARGS__);                                                            \
    } while (0)

extern "C" int hgq_group_norm_fwd(const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, int64_t B,
                                  int64_t S, int C, int G, float eps, int activation, int type, void *workspace, size_t workspace_bytes,
                                  void *stream) {
    int err;
    if (!gn_args_ok(B, S, C, G, activation, type, &err)) return err;
    if (B == 0 || S == 0) return HGQ_OK;
    if (!x || !y || !mean || !rstd) return HGQ_ERR_NULL;
    const size_t size = type == HGQ_TYPE_F32 ? 4 : 2;
    if (!aligned(x, size) || !aligned(y, size) || !aligned(gamma, 4) || !aligned(beta, 4) || !aligned(mean, 4) || !aligned(rstd, 4))
        return HGQ_ERR_ALIGN;
    const SlabPlan plan = gn_plan(x, y, nullptr, B, S, C, G, type, false);
    if (!plan.usable && (!workspace || workspace_bytes < hgq_group_norm_workspace(B, S, C, G, type, 0))) return HGQ_ERR_WORKSPACE;
    if (!aligned(workspace, 4)) return HGQ_ERR_ALIGN;
    if (plan.usable) return gn_slab_fwd(plan, x, gamma, beta, y, mean, rstd, B, S, C, G, eps, activation, type, (cudaStream_t)stream);
    const int vec = gn_vec(x, y, nullptr, C, type);
    GN_DISPATCH(gn_fwd_any, x, gamma, beta, y, mean, rstd, B, S, C, G, eps, activation, (float *)workspace, (cudaStream_t)stream);
}

extern "C" int hgq_group_norm_bwd(const void *gy, const void *x, const float *gamma, const float *beta, const float *mean, const float *rstd,
                                  void *dx, float *dgamma, float *dbeta, int64_t B, int64_t S, int C, int G, int activation, int type,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    int err;
    if (!gn_args_ok(B, S, C, G, activation, type, &err)) return err;
    if ((dgamma == nullptr) != (dbeta == nullptr)) return HGQ_ERR_NULL;
    if (dx == nullptr && dgamma == nullptr) return HGQ_ERR_NULL;
    if (!aligned(dgamma, 4) || !aligned(dbeta, 4)) return HGQ_ERR_ALIGN;
    cudaStream_t st = (cudaStream_t)stream;
    if (B == 0 || S == 0) {
        if (dgamma != nullptr) {
            cudaError_t e = cudaMemsetAsync(dgamma, 0, (size_t)C * sizeof(float), st);
            if (e == cudaSuccess) e = cudaMemsetAsync(dbeta, 0, (size_t)C * sizeof(float), st);
            if (e != cudaSuccess) return (int)e;
        }
        return HGQ_OK;
    }
    if (!gy || !x || !mean || !rstd) return HGQ_ERR_NULL;
    const size_t size = type == HGQ_TYPE_F32 ? 4 : 2;
    if (!aligned(gy, size) || !aligned(x, size) || !aligned(dx, size) || !aligned(gamma, 4) || !aligned(beta, 4) || !aligned(mean, 4) ||
        !aligned(rstd, 4))
        return HGQ_ERR_ALIGN;
    if (!workspace || workspace_bytes < hgq_group_norm_workspace(B, S, C, G, type, 1)) return HGQ_ERR_WORKSPACE;
    if (!aligned(workspace, 4)) return HGQ_ERR_ALIGN;
    float *part = (float *)workspace;
    const SlabPlan plan = gn_plan(gy, x, dx, B, S, C, G, type, true);
    if (plan.usable) {
        if (int e = gn_slab_bwd(plan, gy, x, gamma, beta, mean, rstd, dx, dgamma != nullptr ? part : nullptr, B, S, C, G, activation, type, st))
            return e;
        const int64_t rows = plan.workers * plan.K;
        return dgamma != nullptr ? gn_colsum(part, rows, C, part + rows * 2 * C, dgamma, dbeta, st) : HGQ_OK;
    }
    const int vec = gn_vec(gy, x, dx, C, type);
    float *m = part + gn_part_floats(B, S, C, G, type, true);
    float *scratch = m + 2 * gn_group(B, S, C, 2 * (int)size) * G;
    GN_DISPATCH(gn_bwd_any, gy, x, gamma, beta, mean, rstd, dx, dgamma, dbeta, B, S, C, G, activation, part, m, scratch, st);
}
