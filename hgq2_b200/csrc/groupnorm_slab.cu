// Group normalisation of samples that fit on chip: x (and gy) are read from memory once.
//
// A slab is whole groups of channels of one sample; its rows (positions) are shared by a cluster of K CTAs, and a thread holds R
// packs of VEC neighbouring channels in registers from the one read to the write.  The statistics are two block reductions (mean,
// then centred squares: data whose mean is large against its spread keep their variance), joined over the cluster through
// distributed shared memory in rank order.  Small samples share a CTA.  Registers rather than shared memory hold the data because
// every value is used by the thread that loaded it; what crosses threads is one number a pack (a pack that spans several groups:
// one a channel).
//
// Backward: the CTAs are resident and walk over the samples, so that dgamma and dbeta stay in registers until the end (one row of
// partial sums a CTA, added up in a fixed order by a second launch).  du gamma is kept in fp32 in place of gy between the two uses.
#include <cooperative_groups.h>

#include "groupnorm.cuh"

namespace hgq {

namespace cg = cooperative_groups;

constexpr int kSlabThreads = 256;
constexpr int kSlabWarps = kSlabThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxPairs = 512;  // (sample, group) pairs of a CTA

struct SlabArgs {
    int64_t B, S, items, workers;
    int C, G, Cg, Cs, Gs, slabs, TX, TY, K, subs, rows;
    int width;    // reduction entries of a thread row: TX (one a pack) or TX VEC (one a channel)
    int per_row;  // of them that belong to one group
    FastDiv by_per_row;
};

// Where a thread works: its channels, its sample among the CTA's and its first row.
struct SlabPlace {
    int slab, groups, channels;  // of this slab
    int tx, ty, sub, row, rank;
    int64_t worker;
    bool in;
};

__device__ __forceinline__ SlabPlace slab_place(const SlabArgs &a, int vec) {
    SlabPlace p;
    const int cluster = blockIdx.x / a.K;
    p.rank = blockIdx.x % a.K;
    p.slab = cluster % a.slabs;
    p.worker = cluster / a.slabs;
    p.groups = min(a.Gs, a.G - p.slab * a.Gs);
    p.channels = p.groups * a.Cg;
    p.tx = threadIdx.x % a.TX;
    p.ty = threadIdx.x / a.TX;
    p.in = p.ty < a.TY && p.tx * vec < p.channels;
    if (a.subs > 1) {
        p.sub = p.ty / (int)a.S;
        p.row = p.ty % (int)a.S;
        p.in = p.in && p.sub < a.subs;
    } else {
        p.sub = 0;
        p.row = p.ty;
    }
    return p;
}

// Sums over the (sample of the CTA, group) pairs.  entries: [TY][width] in shared memory, complete; out[pair] = the pair's sum, by a
// power of two of neighbouring lanes each, all pairs at once where they are few.  Every thread of the block calls it.
template <int N>
__device__ __forceinline__ void pair_sums(const float *entries, int stride, float *out, int out_stride, const SlabArgs &a, const SlabPlace &p) {
    const int pairs = a.subs * p.groups;
    const int rows = a.subs > 1 ? (int)a.S : a.TY;
    const int n = rows * a.per_row;
    int lanes = 32;
    while (lanes > 1 && (lanes * pairs > kSlabThreads || lanes > n)) lanes >>= 1;
    const int at_once = kSlabThreads / lanes, l = threadIdx.x % lanes, first = threadIdx.x / lanes;
    for (int base = 0; base < pairs; base += at_once) {
        const int pair = base + first;
        float s[N];
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] = 0.f;
        if (pair < pairs) {
            const int sub = a.subs > 1 ? pair / p.groups : 0, g = pair - sub * p.groups;
            const float *e = entries + (sub * rows) * a.width + g * a.per_row;
            for (int j = l; j < n; j += lanes) {
                const int r = (int)fastdiv((uint32_t)j, a.by_per_row), c = j - r * a.per_row;
#pragma unroll
                for (int k = 0; k < N; ++k) s[k] += e[k * stride + r * a.width + c];
            }
        }
        for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < N; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
        if (pair < pairs && l == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) out[k * out_stride + pair] = s[k];
    }
}

// One thread's contributions (VEC channel sums) into the entries: one a pack or one a channel.
template <int VEC, bool MULTI>
__device__ __forceinline__ void put_entries(float *entries, const float (&v)[VEC], const SlabArgs &a, const SlabPlace &p) {
    if (p.ty >= a.TY) return;
    float *e = entries + p.ty * a.width;
    if (MULTI) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[p.tx * VEC + i] = v[i];
    } else {
        float s = v[0];
#pragma unroll
        for (int i = 1; i < VEC; ++i) s += v[i];
        e[p.tx] = s;
    }
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

template <typename T, int VEC, int R, bool MULTI>
__global__ void __launch_bounds__(kSlabThreads, R * VEC >= 64 ? 2 : (R * VEC >= 32 ? 3 : 4))
    k_gn_slab_fwd(const T *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta, const SlabArgs a, float eps, int act,
                  T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ float entries[kSlabThreads * (MULTI ? VEC : 1)];
    __shared__ float local[2][kMaxPairs], total[2][kMaxPairs];
    const SlabPlace p = slab_place(a, VEC);
    const int c0 = p.slab * a.Cs + p.tx * VEC;
    const int pairs = a.subs * p.groups;
    const float inv_n = 1.f / ((float)a.S * (float)a.Cg);
    float ga[VEC], be[VEC];
    int pair_of[MULTI ? VEC : 1];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        ga[i] = p.in && gamma != nullptr ? gamma[c0 + i] : 1.f;
        be[i] = p.in && beta != nullptr ? beta[c0 + i] : 0.f;
        if (MULTI || i == 0) pair_of[i] = p.in ? p.sub * p.groups + (p.tx * VEC + i) / a.Cg : 0;
    }
    for (int64_t item = p.worker; item < a.items; item += a.workers) {
        const int64_t b = item * a.subs + p.sub;
        const int64_t row = (int64_t)p.rank * a.rows + p.row;
        unsigned mask = 0;
        if (p.in && b < a.B) {
            const int64_t end = a.subs > 1 ? a.S : min(a.S, (int64_t)(p.rank + 1) * a.rows);
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (row + j * a.TY < end && (j == 0 || a.subs == 1)) mask |= 1u << j;
        }
        const int64_t base = (b * a.S + row) * a.C + c0, step = (int64_t)a.TY * a.C;
        Held<T, VEC, R> h;
        h.load(x + base, step, mask);
        float s[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float v[VEC];
            h.values(j, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) s[i] += v[i];
        }
        // mean, then centred squares
        float mu[MULTI ? VEC : 1], rs[MULTI ? VEC : 1];
#pragma unroll
        for (int phase = 0; phase < 2; ++phase) {
            put_entries<VEC, MULTI>(entries, s, a, p);
            __syncthreads();
            pair_sums<1>(entries, 0, local[phase], 0, a, p);
            if (a.K > 1) {
                cg::cluster_group cluster = cg::this_cluster();
                cluster.sync();
                for (int i = threadIdx.x; i < pairs; i += kSlabThreads) {
                    float t = 0.f;
                    for (int k = 0; k < a.K; ++k) t += *cluster.map_shared_rank(&local[phase][i], k);
                    total[phase][i] = t;
                }
            } else {
                __syncthreads();
            }
            const float *sums = a.K > 1 ? total[phase] : local[phase];
            if (a.K > 1) __syncthreads();
            if (phase == 0) {
#pragma unroll
                for (int i = 0; i < (MULTI ? VEC : 1); ++i) mu[i] = sums[pair_of[i]] * inv_n;
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[i] = 0.f;
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (mask >> j & 1) {
                        float v[VEC];
                        h.values(j, v);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            const float d = v[i] - mu[MULTI ? i : 0];
                            s[i] += d * d;
                        }
                    }
            } else {
#pragma unroll
                for (int i = 0; i < (MULTI ? VEC : 1); ++i) rs[i] = 1.f / sqrtf(sums[pair_of[i]] * inv_n + eps);
                if (p.rank == 0)
                    for (int i = threadIdx.x; i < pairs; i += kSlabThreads) {
                        const int sub = i / p.groups;
                        const int64_t bb = item * a.subs + sub;
                        if (bb < a.B) {
                            const int64_t o = bb * a.G + p.slab * a.Gs + (i - sub * p.groups);
                            mean_out[o] = (a.K > 1 ? total[0][i] : local[0][i]) * inv_n;
                            rstd_out[o] = 1.f / sqrtf(sums[i] * inv_n + eps);
                        }
                    }
            }
        }
        GN_FOR_ACT(act, {
            _Pragma("unroll") for (int j = 0; j < R; ++j) if (mask >> j & 1) {
                float v[VEC];
                h.values(j, v);
                _Pragma("unroll") for (int i = 0; i < VEC; ++i) {
                    const int m = MULTI ? i : 0;
                    v[i] = act_value<T, ACT>((v[i] - mu[m]) * (rs[m] * ga[i]) + be[i]);
                }
                store_pack<T, VEC>(y + base + j * step, v);
            }
        })
    }
    if (a.K > 1) cg::this_cluster().sync();  // no CTA leaves while another may still read its sums
}

template <typename T, int VEC, int R, bool MULTI>
__global__ void __launch_bounds__(kSlabThreads, 2)
    k_gn_slab_bwd(const T *__restrict__ gy, const T *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta,
                  const float *__restrict__ mean, const float *__restrict__ rstd, const SlabArgs a, int act, T *__restrict__ dx,
                  float *__restrict__ part) {
    constexpr int kEntries = kSlabThreads * (MULTI ? VEC : 1);
    __shared__ float entries[2 * kEntries];
    __shared__ float local[2][2 * kMaxPairs], total[2][2 * kMaxPairs];
    __shared__ float acc[2 * VEC][kSlabThreads];  // du and du xhat of this thread's channels, over all of the CTA's samples
    const SlabPlace p = slab_place(a, VEC);
    const int c0 = p.slab * a.Cs + p.tx * VEC;
    const int pairs = a.subs * p.groups;
    const float inv_n = 1.f / ((float)a.S * (float)a.Cg);
    float ga[VEC], be[VEC];
    int pair_of[MULTI ? VEC : 1], group_of[MULTI ? VEC : 1];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        ga[i] = p.in && gamma != nullptr ? gamma[c0 + i] : 1.f;
        be[i] = p.in && beta != nullptr ? beta[c0 + i] : 0.f;
        acc[i][threadIdx.x] = acc[VEC + i][threadIdx.x] = 0.f;
        if (MULTI || i == 0) {
            group_of[i] = p.in ? (p.tx * VEC + i) / a.Cg : 0;
            pair_of[i] = (p.in ? p.sub : 0) * p.groups + group_of[i];
        }
    }
    int turn = 0;
    for (int64_t item = p.worker; item < a.items; item += a.workers, turn ^= 1) {
        const int64_t b = item * a.subs + p.sub;
        const int64_t row = (int64_t)p.rank * a.rows + p.row;
        unsigned mask = 0;
        float mu[MULTI ? VEC : 1], rs[MULTI ? VEC : 1];
#pragma unroll
        for (int i = 0; i < (MULTI ? VEC : 1); ++i) mu[i] = rs[i] = 0.f;
        if (p.in && b < a.B) {
            const int64_t end = a.subs > 1 ? a.S : min(a.S, (int64_t)(p.rank + 1) * a.rows);
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (row + j * a.TY < end && (j == 0 || a.subs == 1)) mask |= 1u << j;
#pragma unroll
            for (int i = 0; i < (MULTI ? VEC : 1); ++i) {
                const int64_t o = b * a.G + p.slab * a.Gs + group_of[i];
                mu[i] = mean[o];
                rs[i] = rstd[o];
            }
        }
        const int64_t base = (b * a.S + row) * a.C + c0, step = (int64_t)a.TY * a.C;
        Held<T, VEC, R> h, hg;
        h.load(x + base, step, mask);
        hg.load(gy + base, step, mask);
        float t[R][VEC], du_[VEC], dux[VEC];  // t: du gamma
#pragma unroll
        for (int i = 0; i < VEC; ++i) du_[i] = dux[i] = 0.f;
        GN_FOR_ACT(act, {
            _Pragma("unroll") for (int j = 0; j < R; ++j) if (mask >> j & 1) {
                float v[VEC], d[VEC];
                h.values(j, v);
                hg.values(j, d);
                _Pragma("unroll") for (int i = 0; i < VEC; ++i) {
                    const int m = MULTI ? i : 0;
                    const float xh = (v[i] - mu[m]) * rs[m];
                    const float du = d[i] * act_slope<T, ACT>(xh * ga[i] + be[i]);
                    du_[i] += du;
                    dux[i] += du * xh;
                    t[j][i] = du * ga[i];
                }
            }
        })
        float w1[VEC], w2[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            acc[i][threadIdx.x] += du_[i];
            acc[VEC + i][threadIdx.x] += dux[i];
            w1[i] = du_[i] * ga[i];
            w2[i] = dux[i] * ga[i];
        }
        if (dx == nullptr) continue;  // the parameters' gradients alone
        put_entries<VEC, MULTI>(entries, w1, a, p);
        put_entries<VEC, MULTI>(entries + kEntries, w2, a, p);
        __syncthreads();
        pair_sums<2>(entries, kEntries, local[turn], kMaxPairs, a, p);
        const float *sums = local[turn];
        if (a.K > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
            for (int i = threadIdx.x; i < pairs; i += kSlabThreads) {
                float t1 = 0.f, t2 = 0.f;
                for (int k = 0; k < a.K; ++k) {
                    t1 += *cluster.map_shared_rank(&local[turn][i], k);
                    t2 += *cluster.map_shared_rank(&local[turn][kMaxPairs + i], k);
                }
                total[turn][i] = t1;
                total[turn][kMaxPairs + i] = t2;
            }
            sums = total[turn];
        }
        __syncthreads();
        float m1[MULTI ? VEC : 1], m2[MULTI ? VEC : 1];
#pragma unroll
        for (int i = 0; i < (MULTI ? VEC : 1); ++i) {
            m1[i] = sums[pair_of[i]] * inv_n;
            m2[i] = sums[kMaxPairs + pair_of[i]] * inv_n;
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (mask >> j & 1) {
                float v[VEC];
                h.values(j, v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const int m = MULTI ? i : 0;
                    const float xh = (v[i] - mu[m]) * rs[m];
                    v[i] = rs[m] * (t[j][i] - m1[m] - xh * m2[m]);
                }
                store_pack<T, VEC>(dx + base + j * step, v);
            }
    }
    if (part != nullptr) {
        // this CTA's sums per channel, over its thread rows
        float *out = part + (p.worker * a.K + p.rank) * 2 * a.C;
        __syncthreads();
        for (int c = threadIdx.x; c < p.channels; c += kSlabThreads) {
            float s1 = 0.f, s2 = 0.f;
            for (int r = 0; r < a.TY; ++r) {
                s1 += acc[c % VEC][r * a.TX + c / VEC];
                s2 += acc[VEC + c % VEC][r * a.TX + c / VEC];
            }
            out[p.slab * a.Cs + c] = s1;
            out[a.C + p.slab * a.Cs + c] = s2;
        }
    }
    if (a.K > 1) cg::this_cluster().sync();
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// Packs a thread holds: enough of them that a CTA has 16 to 32 KB of a tensor in flight.
static int slab_most(int type, int vec, bool backward) {
    const int size = type == HGQ_TYPE_F32 ? 4 : 2;
    if (vec * size < 16) return 16;  // narrow packs: many of them
    return backward && type != HGQ_TYPE_F32 ? 4 : 8;
}

SlabPlan gn_slab_plan(int64_t B, int64_t S, int C, int G, int type, int vec, bool backward) {
    SlabPlan p{};
    const int Cg = C / G, size = type == HGQ_TYPE_F32 ? 4 : 2;
    const int most = slab_most(type, vec, backward);
    p.vec = vec;
    p.multi = Cg % vec != 0;
    // whole groups whose channels are whole packs
    int unit = Cg;
    while (unit % vec != 0) unit += Cg;  // at most vec groups
    if (C % unit != 0 || unit / vec > kSlabThreads) return p;
    // Slabs as wide as 128 threads allow (wide rows are read whole), narrower where the rows of a slab would not fit, but no
    // narrower than the 64 bytes that keep memory sectors whole unless the channels are fewer.
    int units = C / unit;
    int per = units;
    while (per > 1 && (per * unit / vec > 128 || per * unit / Cg > kMaxPairs)) per = (per + 1) / 2;
    if (per * unit / Cg > kMaxPairs) return p;
    for (;; per = (per + 1) / 2) {
        p.Cs = per * unit;
        p.TX = p.Cs / vec;
        p.TY = kSlabThreads / p.TX;
        const int64_t fits = (int64_t)p.TY * most * kMaxCluster;
        if (S <= fits) break;
        if (per == 1 || ((per + 1) / 2) * unit * size < 64) return p;
    }
    p.Gs = p.Cs / Cg;
    p.slabs = (G + p.Gs - 1) / p.Gs;
    p.subs = 1;
    p.K = 1;
    if (2 * S <= p.TY) {
        p.subs = p.TY / (int)S;
        if (p.subs > B) p.subs = (int)B;
        if (p.subs > kMaxPairs / p.Gs) p.subs = kMaxPairs / p.Gs;
        if (p.subs < 1) p.subs = 1;
    }
    const int64_t packs = (S + p.TY - 1) / p.TY;  // a thread would hold with one CTA
    while (packs > (int64_t)most * p.K) p.K <<= 1;
    p.rows = (int)((S + p.K - 1) / p.K);
    const int need = (p.rows + p.TY - 1) / p.TY;
    p.R = need <= 1 ? 1 : (need <= 4 && most != 16 ? 4 : most);
    p.items = (B + p.subs - 1) / p.subs;
    if (p.items * p.slabs * p.K > INT32_MAX) return p;
    p.workers = p.items;
    if (backward) {
        // resident CTAs: two an SM; a cluster's CTAs are placed together
        int64_t n = (int64_t)num_sms() * 2 / ((int64_t)p.K * p.slabs);
        if (n < 1) n = 1;
        if (p.workers > n) p.workers = n;
    }
    p.usable = true;
    return p;
}

static SlabArgs slab_args(const SlabPlan &p, int64_t B, int64_t S, int C, int G) {
    SlabArgs a{};
    a.B = B, a.S = S, a.items = p.items, a.workers = p.workers;
    a.C = C, a.G = G, a.Cg = C / G, a.Cs = p.Cs, a.Gs = p.Gs, a.slabs = p.slabs, a.TX = p.TX, a.TY = p.TY, a.K = p.K, a.subs = p.subs,
    a.rows = p.rows;
    a.width = p.multi ? p.TX * p.vec : p.TX;
    a.per_row = p.multi ? a.Cg : a.Cg / p.vec;
    a.by_per_row = make_fastdiv((uint32_t)a.per_row);
    return a;
}

template <typename... Params, typename... Args>
static int launch_clusters(void (*kernel)(Params...), int64_t ctas, int K, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kSlabThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)K;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = K > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return (int)e;
    }
    return check_launch();
}

template <typename T, int VEC, int R>
static int slab_fwd(const SlabPlan &p, const SlabArgs &a, const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd,
                    float eps, int act, cudaStream_t st) {
    const int64_t ctas = p.workers * p.slabs * p.K;
    if (VEC > 1 && p.multi)
        return launch_clusters(k_gn_slab_fwd<T, VEC, R, true>, ctas, p.K, st, (const T *)x, gamma, beta, a, eps, act, (T *)y, mean, rstd);
    return launch_clusters(k_gn_slab_fwd<T, VEC, R, false>, ctas, p.K, st, (const T *)x, gamma, beta, a, eps, act, (T *)y, mean, rstd);
}

template <typename T, int VEC, int R>
static int slab_bwd(const SlabPlan &p, const SlabArgs &a, const void *gy, const void *x, const float *gamma, const float *beta, const float *mean,
                    const float *rstd, int act, void *dx, float *part, cudaStream_t st) {
    const int64_t ctas = p.workers * p.slabs * p.K;
    if (VEC > 1 && p.multi)
        return launch_clusters(k_gn_slab_bwd<T, VEC, R, true>, ctas, p.K, st, (const T *)gy, (const T *)x, gamma, beta, mean, rstd, a, act,
                               (T *)dx, part);
    return launch_clusters(k_gn_slab_bwd<T, VEC, R, false>, ctas, p.K, st, (const T *)gy, (const T *)x, gamma, beta, mean, rstd, a, act, (T *)dx,
                           part);
}

#define SLAB_DISPATCH(FN, FULL_MOST, ...)                                              \
    do {                                                                               \
        if (type == HGQ_TYPE_F32) {                                                    \
            if (p.vec == 4 && p.R == 1) return FN<float, 4, 1>(__VA_ARGS__);           \
            if (p.vec == 4 && p.R == 4) return FN<float, 4, 4>(__VA_ARGS__);           \
            if (p.vec == 4) return FN<float, 4, 8>(__VA_ARGS__);                       \
            if (p.vec == 2 && p.R == 1) return FN<float, 2, 1>(__VA_ARGS__);           \
            if (p.vec == 2) return FN<float, 2, 16>(__VA_ARGS__);                      \
            if (p.R == 1) return FN<float, 1, 1>(__VA_ARGS__);                         \
            return FN<float, 1, 16>(__VA_ARGS__);                                      \
        }                                                                              \
        if (type == HGQ_TYPE_BF16) SLAB_HALF(FN, FULL_MOST, __nv_bfloat16, __VA_ARGS__); \
        SLAB_HALF(FN, FULL_MOST, __half, __VA_ARGS__);                                 \
    } while (0)

#define SLAB_HALF(FN, FULL_MOST, T, ...)                                 \
    do {                                                                 \
        if (p.vec == 8 && p.R == 1) return FN<T, 8, 1>(__VA_ARGS__);     \
        if (p.vec == 8 && p.R == 4) return FN<T, 8, 4>(__VA_ARGS__);     \
        if (p.vec == 8) return FN<T, 8, FULL_MOST>(__VA_ARGS__);         \
        if (p.vec == 2 && p.R == 1) return FN<T, 2, 1>(__VA_ARGS__);     \
        if (p.vec == 2) return FN<T, 2, 16>(__VA_ARGS__);                \
        if (p.R == 1) return FN<T, 1, 1>(__VA_ARGS__);                   \
        return FN<T, 1, 16>(__VA_ARGS__);                                \
    } while (0)

int gn_slab_fwd(const SlabPlan &p, const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, int64_t B,
                int64_t S, int C, int G, float eps, int act, int type, cudaStream_t st) {
    const SlabArgs a = slab_args(p, B, S, C, G);
    SLAB_DISPATCH(slab_fwd, 8, p, a, x, gamma, beta, y, mean, rstd, eps, act, st);
}

int gn_slab_bwd(const SlabPlan &p, const void *gy, const void *x, const float *gamma, const float *beta, const float *mean,
                const float *rstd, void *dx, float *part, int64_t B, int64_t S, int C, int G, int act, int type, cudaStream_t st) {
    const SlabArgs a = slab_args(p, B, S, C, G);
    SLAB_DISPATCH(slab_bwd, 4, p, a, gy, x, gamma, beta, mean, rstd, act, dx, part, st);
}

}  // namespace hgq
