// Group normalisation of samples that fit on chip: x (and gy) are read from memory once.
//
// A slab is whole groups of channels of one sample; its rows (positions) are shared by a cluster of K CTAs, and a thread holds R
// packs of VEC neighbouring channels in registers from the one read to the write.  The statistics are two block reductions (mean,
// then centred squares: data whose mean is large against its spread keep their variance), joined over the cluster through
// distributed shared memory in rank order.  Small samples share a CTA.  Registers rather than shared memory hold the data because
// every value is used by the thread that loaded it; what crosses threads is one number a pack (one a group that the pack touches).
// The CTAs are resident and walk over the samples.
//
// Backward: dgamma and dbeta add up in shared memory, a place for each thread, until the end (one row of partial sums a CTA, added
// up in a fixed order by a second launch).  du gamma is kept in fp32 in place of gy between its two uses.
//
// What bounds it: forward, memory for fp32 ([4096, 30, 30, 16] with SiLU 0.085 ms = 0.84 of the 6.57 TB/s copy rate; [8192, 64, 64]
// 0.051 ms = 0.80), latency and issue slots for bf16 ([8192, 64, 64] with ReLU 0.031 ms = 0.67).  A total costs what its threads
// cost, so a sample takes as few threads as hold it (0.069 -> 0.035 ms there), and the next sample's packs are fetched while this
// one's totals are taken.  Backward: du gamma in registers leaves two CTAs an SM, 0.175 and 0.089 ms for the fp32 shapes (0.62 and
// 0.69).  Two CTAs share a sample that one cannot hold; four or eight wait for one another longer than the second read of the other
// kernels takes ([256, 1024, 128] bf16: 0.104 ms with eight, 0.062 with two or none).  x staged in shared memory for its second use
// in the backward pass made the registers spill more (0.187 -> 0.189 ms) and was left out.  As it is, 53 of the 144 variants spill, most of
// them those with a number a channel (packs that groups do not nest with; up to 224 bytes, fp32 backward) and those of narrow packs.
#include <cooperative_groups.h>

#include "groupnorm.cuh"

namespace hgq {

namespace cg = cooperative_groups;

constexpr int kSlabThreads = kThreads;
constexpr int kSlabWarps = kSlabThreads / 32;
constexpr int kMaxCluster = 2;
constexpr int kMaxPairs = 512;  // (sample, group) pairs of a CTA

// Channel counts that packs do not divide: q rows in a row are taken as one of q C channels, which packs do divide; S and C are
// those of the joined rows, `channels` the real count.
struct SlabArgs {
    int64_t B, S, items, workers;
    float inv_n;  // 1 / (values of a group)
    int channels, q;
    int C, G, Cg, Cs, Gs, slabs, TX, TY, K, subs, rows;
    int TYs;  // thread rows of one sample: TY / subs
    int per_row;  // neighbouring threads of a row that belong to one group (one a pack), or 1
    // Totals over a (sample, group).  `bits`: all extents are powers of two, so that the threads of one total differ exactly in
    // certain bits of their index: those of lane_bits meet in shuffles, those of warp_bits through shared memory.
    bool bits;
    unsigned lane_bits, warp_bits;
    // Otherwise: entries in shared memory, [TY][width]; a row has q runs (one every `channels`) of `run` entries for a group.
    int width, run, per_group;  // per_group = q run
    FastDiv by_per_group, by_run;
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
    p.channels = a.q > 1 ? a.C : p.groups * a.Cg;
    p.tx = threadIdx.x % a.TX;
    p.ty = threadIdx.x / a.TX;
    p.in = p.ty < a.TY && p.tx * vec < p.channels;
    p.sub = a.subs > 1 ? p.ty / a.TYs : 0;
    p.row = a.subs > 1 ? p.ty - p.sub * a.TYs : p.ty;
    p.in = p.in && p.sub < a.subs;
    return p;
}

// What a CTA needs to add up N sets of NG numbers a thread over the threads of each (sample, group).
template <int NG, int N>
struct SumSpace {
    float entries[N * NG * kSlabThreads];
    float pair[2][N][kMaxPairs];  // by turns
    float all[N][kMaxPairs];      // over the cluster
};

// v: in, a thread's numbers (one a group that its pack touches; NG == VEC: one a channel), out, the totals of their groups, over the
// cluster.  pair_of: the (sample of the CTA, group) of each.  Every thread of the block calls it, `turn` alternating.
template <int NG, int N>
__device__ __forceinline__ void group_totals(float (&v)[N][NG], SumSpace<NG, N> &sh, int turn, const int (&pair_of)[NG], const SlabArgs &a,
                                             const SlabPlace &p) {
    const int tid = threadIdx.x;
    if (a.bits) {
#pragma unroll
        for (unsigned o = 1; o < 32; o <<= 1)
            if (a.lane_bits & o)
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int i = 0; i < NG; ++i) v[k][i] += __shfl_xor_sync(0xffffffffu, v[k][i], o);
        if (a.warp_bits != 0) {
            float *e = sh.entries;
            if ((tid & a.lane_bits) == 0)
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int i = 0; i < NG; ++i) e[(k * NG + i) * kSlabThreads + tid] = v[k][i];
            __syncthreads();
            const int base = tid & ~(int)(a.lane_bits | a.warp_bits);
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
                for (int i = 0; i < NG; ++i) v[k][i] = 0.f;
            if (a.warp_bits == kSlabThreads - 32) {  // all warps: the same sums in the same order, unrolled
#pragma unroll
                for (int w = 0; w < kSlabWarps; ++w)
#pragma unroll
                    for (int k = 0; k < N; ++k)
#pragma unroll
                        for (int i = 0; i < NG; ++i) v[k][i] += e[(k * NG + i) * kSlabThreads + base + w * 32];
            } else {
                unsigned w = 0;  // the subsets of warp_bits in ascending order
                do {
#pragma unroll
                    for (int k = 0; k < N; ++k)
#pragma unroll
                        for (int i = 0; i < NG; ++i) v[k][i] += e[(k * NG + i) * kSlabThreads + (base | w)];
                    w = (w - a.warp_bits) & a.warp_bits;
                } while (w != 0);
            }
        }
        if (a.K > 1 && p.in && (tid & (a.lane_bits | a.warp_bits)) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
                for (int i = 0; i < NG; ++i) sh.pair[turn][k][pair_of[i]] = v[k][i];
        if (a.K == 1) {
            if (a.warp_bits != 0) __syncthreads();  // the entries are free again
            return;
        }
    } else {
        const int pairs = a.subs * p.groups, rows = a.TYs, n = rows * a.per_group;
        if (p.ty < a.TY)
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
                for (int i = 0; i < NG; ++i) sh.entries[k * NG * kSlabThreads + p.ty * a.width + p.tx * NG + i] = v[k][i];
        __syncthreads();
        // a power of two of neighbouring lanes for each pair, all pairs at once where they are few
        int lanes = 32;
        while (lanes > 1 && (lanes * pairs > kSlabThreads || lanes > n)) lanes >>= 1;
        const int at_once = kSlabThreads / lanes, l = tid & (lanes - 1), first = tid / lanes;
        for (int base = 0; base < pairs; base += at_once) {
            const int pair = base + first;
            float s[N];
#pragma unroll
            for (int k = 0; k < N; ++k) s[k] = 0.f;
            if (pair < pairs) {
                const int sub = a.subs > 1 ? pair / p.groups : 0, g = pair - sub * p.groups;
                const float *e = sh.entries + (sub * rows) * a.width + g * a.run;
                for (int j = l; j < n; j += lanes) {
                    const int r = (int)fastdiv((uint32_t)j, a.by_per_group);
                    int c = j - r * a.per_group;
                    if (a.q > 1) c += (int)fastdiv((uint32_t)c, a.by_run) * (a.channels - a.run);
#pragma unroll
                    for (int k = 0; k < N; ++k) s[k] += e[k * NG * kSlabThreads + r * a.width + c];
                }
            }
            for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
                for (int k = 0; k < N; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
            if (pair < pairs && l == 0)
#pragma unroll
                for (int k = 0; k < N; ++k) sh.pair[turn][k][pair] = s[k];
        }
    }
    if (a.K > 1) {
        // the CTAs' totals in rank order; each CTA's of this turn stay until the next turn's barrier
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int pairs = a.subs * p.groups;
        for (int i = tid; i < pairs; i += kSlabThreads)
#pragma unroll
            for (int k = 0; k < N; ++k) {
                float t = 0.f;
                for (int r = 0; r < a.K; ++r) t += *cluster.map_shared_rank(&sh.pair[turn][k][i], r);
                sh.all[k][i] = t;
            }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < NG; ++i) v[k][i] = a.K > 1 ? sh.all[k][pair_of[i]] : sh.pair[turn][k][pair_of[i]];
}

// The channels of a pack as the NG groups they belong to.
template <int VEC, int NG>
__device__ __forceinline__ void join_channels(const float (&c)[VEC], float (&g)[NG]) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        g[i] = c[i * (VEC / NG)];
#pragma unroll
        for (int j = 1; j < VEC / NG; ++j) g[i] += c[i * (VEC / NG) + j];
    }
}

// CTAs an SM, by the registers that the held packs take.
constexpr int slab_fwd_ctas(int values, bool ahead) { return ahead ? (values >= 32 ? 2 : 3) : (values >= 64 ? 2 : (values >= 32 ? 3 : 4)); }

template <typename T, int VEC, int R, int NG, bool AHEAD>
__global__ void __launch_bounds__(kSlabThreads, slab_fwd_ctas(R * VEC, AHEAD))
    k_gn_slab_fwd(const T *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta, const SlabArgs a, float eps, int act,
                  T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    constexpr int W = VEC / NG;  // channels of a pack in one group
    __shared__ SumSpace<NG, 1> sh;
    const SlabPlace p = slab_place(a, VEC);
    const int c0 = p.slab * a.Cs + p.tx * VEC;
    const float inv_n = a.inv_n;
    float ga[VEC], be[VEC];
    int pair_of[NG], group_of[NG];
    unsigned writes = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int c = a.q > 1 ? (c0 + i) % a.channels : c0 + i;
        ga[i] = p.in && gamma != nullptr ? gamma[c] : 1.f;
        be[i] = p.in && beta != nullptr ? beta[c] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int c = p.tx * VEC + i * W;
        group_of[i] = p.in ? (a.q > 1 ? c % a.channels : c) / a.Cg : 0;
        pair_of[i] = (p.in ? p.sub : 0) * p.groups + group_of[i];
        // the first thread of each (sample, group) writes its statistics: the first row's first pack of it
        if (p.in && p.rank == 0 && p.row == 0 && c < a.channels && c % a.Cg == 0) writes |= 1u << i;
    }
    const int64_t step = (int64_t)a.TYs * a.C, end = min(a.S, (int64_t)(p.rank + 1) * a.rows);
    const int64_t row = (int64_t)p.rank * a.rows + p.row;
    unsigned rows_mask = 0;
#pragma unroll
    for (int j = 0; j < R; ++j)
        if (row + j * a.TYs < end) rows_mask |= 1u << j;
    using H = Held<T, VEC, R>;
    extern __shared__ __align__(16) unsigned char stage[];
    auto mask_of = [&](int64_t item) { return p.in && item < a.items && item * a.subs + p.sub < a.B ? rows_mask : 0u; };
    auto base_of = [&](int64_t item) { return ((item * a.subs + p.sub) * a.S + row) * a.C + c0; };
    if (AHEAD) H::fetch(stage, x + base_of(p.worker), step, mask_of(p.worker));
    for (int64_t item = p.worker; item < a.items; item += a.workers) {
        const int64_t b = item * a.subs + p.sub;
        const unsigned mask = mask_of(item);
        const int64_t base = base_of(item);
        H h;
        if (AHEAD) {
            H::arrived();
            h.take(stage, mask);
        } else {
            h.load(x + base, step, mask);
        }
        float s[VEC], mu[1][NG], rs[1][NG];
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float v[VEC];
            h.values(j, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) s[i] += v[i];
        }
        join_channels<VEC, NG>(s, mu[0]);
        // every value has been used by now: the places are free for the next sample
        if (AHEAD) H::fetch(stage, x + base_of(item + a.workers), step, mask_of(item + a.workers));
        group_totals<NG, 1>(mu, sh, 0, pair_of, a, p);
#pragma unroll
        for (int i = 0; i < NG; ++i) mu[0][i] *= inv_n;
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (mask >> j & 1) {
                float v[VEC];
                h.values(j, v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = v[i] - mu[0][i / W];
                    s[i] += d * d;
                }
            }
        join_channels<VEC, NG>(s, rs[0]);
        group_totals<NG, 1>(rs, sh, 1, pair_of, a, p);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            rs[0][i] = rsqrtf(rs[0][i] * inv_n + eps);
            if ((writes >> i & 1) && b < a.B) {
                const int64_t o = b * a.G + p.slab * a.Gs + group_of[i];
                mean_out[o] = mu[0][i];
                rstd_out[o] = rs[0][i];
            }
        }
        GN_FOR_ACT(act, {
            _Pragma("unroll") for (int j = 0; j < R; ++j) if (mask >> j & 1) {
                float v[VEC];
                h.values(j, v);
                _Pragma("unroll") for (int i = 0; i < VEC; ++i)
                    v[i] = act_value<T, ACT>((v[i] - mu[0][i / W]) * (rs[0][i / W] * ga[i]) + be[i]);
                store_pack<T, VEC>(y + base + j * step, v);
            }
        })
    }
    if (a.K > 1) cg::this_cluster().sync();  // no CTA leaves while another may still read its sums
}

template <typename T, int VEC, int R, int NG>
__global__ void __launch_bounds__(kSlabThreads, 2)
    k_gn_slab_bwd(const T *__restrict__ gy, const T *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta,
                  const float *__restrict__ mean, const float *__restrict__ rstd, const SlabArgs a, int act, T *__restrict__ dx,
                  float *__restrict__ part) {
    constexpr int W = VEC / NG;
    __shared__ SumSpace<NG, 2> sh;
    __shared__ float acc[2 * VEC][kSlabThreads];  // du and du xhat of this thread's channels, over all of the CTA's samples
    const SlabPlace p = slab_place(a, VEC);
    const int c0 = p.slab * a.Cs + p.tx * VEC;
    const float inv_n = a.inv_n;
    float ga[VEC], be[VEC];
    int pair_of[NG], group_of[NG];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int c = a.q > 1 ? (c0 + i) % a.channels : c0 + i;
        ga[i] = p.in && gamma != nullptr ? gamma[c] : 1.f;
        be[i] = p.in && beta != nullptr ? beta[c] : 0.f;
        acc[i][threadIdx.x] = acc[VEC + i][threadIdx.x] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int c = p.tx * VEC + i * W;
        group_of[i] = p.in ? (a.q > 1 ? c % a.channels : c) / a.Cg : 0;
        pair_of[i] = (p.in ? p.sub : 0) * p.groups + group_of[i];
    }
    const int64_t step = (int64_t)a.TYs * a.C, end = min(a.S, (int64_t)(p.rank + 1) * a.rows);
    const int64_t row = (int64_t)p.rank * a.rows + p.row;
    unsigned rows_mask = 0;
#pragma unroll
    for (int j = 0; j < R; ++j)
        if (row + j * a.TYs < end) rows_mask |= 1u << j;
    int turn = 0;
    for (int64_t item = p.worker; item < a.items; item += a.workers, turn ^= 1) {
        const int64_t b = item * a.subs + p.sub;
        const bool in = p.in && b < a.B;
        const unsigned mask = in ? rows_mask : 0;
        const int64_t base = (b * a.S + row) * a.C + c0;
        Held<T, VEC, R> h, hg;
        h.load(x + base, step, mask);
        hg.load(gy + base, step, mask);
        float mu[NG], rs[NG];
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int64_t o = b * a.G + p.slab * a.Gs + group_of[i];
            mu[i] = in ? mean[o] : 0.f;
            rs[i] = in ? rstd[o] : 0.f;
        }
        float t[R][VEC], du_[VEC], dux[VEC];  // t: du gamma
#pragma unroll
        for (int i = 0; i < VEC; ++i) du_[i] = dux[i] = 0.f;
        GN_FOR_ACT(act, {
            _Pragma("unroll") for (int j = 0; j < R; ++j) if (mask >> j & 1) {
                float v[VEC], d[VEC];
                h.values(j, v);
                hg.values(j, d);
                _Pragma("unroll") for (int i = 0; i < VEC; ++i) {
                    const float xh = (v[i] - mu[i / W]) * rs[i / W];
                    const float du = d[i] * act_slope<T, ACT>(xh * ga[i] + be[i]);
                    du_[i] += du;
                    dux[i] += du * xh;
                    t[j][i] = du * ga[i];
                }
            }
        })
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            acc[i][threadIdx.x] += du_[i];
            acc[VEC + i][threadIdx.x] += dux[i];
            du_[i] *= ga[i];
            dux[i] *= ga[i];
        }
        if (dx == nullptr) continue;  // the parameters' gradients alone
        float m[2][NG];
        join_channels<VEC, NG>(du_, m[0]);
        join_channels<VEC, NG>(dux, m[1]);
        group_totals<NG, 2>(m, sh, turn, pair_of, a, p);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            m[0][i] *= inv_n;
            m[1][i] *= inv_n;
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (mask >> j & 1) {
                float v[VEC];
                h.values(j, v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = (v[i] - mu[i / W]) * rs[i / W];
                    v[i] = rs[i / W] * (t[j][i] - m[0][i / W] - xh * m[1][i / W]);
                }
                store_pack<T, VEC>(dx + base + j * step, v);
            }
    }
    if (part != nullptr) {
        // this CTA's sums per channel, over its thread rows
        float *out = part + (p.worker * a.K + p.rank) * 2 * a.channels;
        __syncthreads();
        const int real = a.q > 1 ? a.channels : p.channels;
        for (int c = threadIdx.x; c < real; c += kSlabThreads) {
            float s1 = 0.f, s2 = 0.f;
            for (int k = c; k < p.channels; k += real)
                for (int r = 0; r < a.TY; ++r) {
                    s1 += acc[k % VEC][r * a.TX + k / VEC];
                    s2 += acc[VEC + k % VEC][r * a.TX + k / VEC];
                }
            out[p.slab * a.Cs + c] = s1;
            out[a.channels + p.slab * a.Cs + c] = s2;
        }
    }
    if (a.K > 1) cg::this_cluster().sync();
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// Packs of one tensor that a thread holds: usually (what leaves two or three CTAs an SM), and at most, where that saves a cluster.
static void slab_held(int type, int vec, bool backward, int &usual, int &most) {
    const bool half = type != HGQ_TYPE_F32;
    const int bytes = vec * (half ? 2 : 4);
    if (bytes == 16) {
        usual = backward && half ? 4 : 8;
        most = backward || half ? usual : 16;
    } else {
        usual = most = half && vec == 4 ? 8 : 16;  // narrow packs: many of them
    }
}

SlabPlan gn_slab_plan(int64_t B, int64_t S, int C, int G, int type, int vec, bool backward) {
    SlabPlan p{};
    p.q = 1;
    while ((int64_t)p.q * C % vec != 0) p.q <<= 1;  // vec is a power of two
    if (S % p.q != 0 || (p.q > 1 && (int64_t)p.q * C / vec > kSlabThreads)) return p;
    const int Cg = C / G, size = type == HGQ_TYPE_F32 ? 4 : 2;
    int usual, most;
    slab_held(type, vec, backward, usual, most);
    p.vec = vec;
    p.groups_of_pack = p.q > 1 ? vec : (Cg % vec == 0 ? 1 : (vec % Cg == 0 ? vec / Cg : vec));
    if (p.q == 1 && Cg > kSlabThreads * vec) return p;
    // whole groups whose channels are whole packs
    S /= p.q;
    C *= p.q;
    int unit = p.q > 1 ? C : Cg;
    while (unit % vec != 0) unit += Cg;  // at most vec groups
    if (C % unit != 0 || unit / vec > kSlabThreads) return p;
    // Slabs as wide as 128 threads allow (wide rows are read whole), narrower where the rows of a slab would not fit, but no
    // narrower than the 64 bytes that keep memory sectors whole unless the channels are fewer.
    int units = C / unit;
    int per = units;
    while (per > 1 && (per * unit / vec > 128 || per * unit / Cg > kMaxPairs)) per = (per + 1) / 2;
    if (per * unit / Cg / p.q > kMaxPairs) return p;
    for (;; per = (per + 1) / 2) {
        p.Cs = per * unit;
        p.TX = p.Cs / vec;
        p.TY = kSlabThreads / p.TX;
        const int64_t fits = (int64_t)p.TY * most * kMaxCluster;
        if (S <= fits) break;
        if (per == 1 || ((per + 1) / 2) * unit * size < 64) return p;
    }
    p.Gs = p.Cs / Cg / p.q;
    p.slabs = (G + p.Gs - 1) / p.Gs;
    // As few thread rows for a sample as hold it (what a total costs is a matter of threads, not of values): the CTA's others take
    // other samples, if there are enough of them to give every SM two CTAs.
    p.subs = 1;
    p.K = 1;
    p.TYs = p.TY;
    if (S <= (int64_t)p.TY * usual) {
        int rows = 1;
        while ((int64_t)rows * usual < S) rows <<= 1;
        while (rows < p.TY && (B * rows < (int64_t)num_sms() * 2 * p.TY || p.TY / rows > kMaxPairs / p.Gs)) rows <<= 1;
        if (2 * rows <= p.TY) {
            p.TYs = rows;
            p.subs = p.TY / rows;
            if (p.subs > B) p.subs = (int)B;
        }
    }
    const int64_t packs = (S + p.TYs - 1) / p.TYs;  // a thread would hold with one CTA
    while (packs > (int64_t)most * p.K) p.K <<= 1;
    p.rows = (int)((S + p.K - 1) / p.K);
    const int need = (p.rows + p.TYs - 1) / p.TYs;
    if (vec * size >= 8 && vec >= 4) p.R = need <= 1 ? 1 : (need <= 4 ? 4 : (need <= 8 ? 8 : 16));
    else p.R = need <= 1 ? 1 : 16;
    p.items = (B + p.subs - 1) / p.subs;
    if (p.items * p.slabs * p.K > INT32_MAX) return p;
    // resident CTAs, by their registers: what a CTA sets up once (places, scale and offset) is spread over its samples
    p.ahead = !backward && p.K == 1 && vec * size == 16;
    int64_t n = (int64_t)num_sms() * (backward ? 2 : slab_fwd_ctas(p.R * vec, p.ahead)) / ((int64_t)p.K * p.slabs);
    if (n < 1) n = 1;
    p.workers = p.items < n ? p.items : n;
    p.usable = true;
    return p;
}

static SlabArgs slab_args(const SlabPlan &p, int64_t B, int64_t S, int C, int G) {
    SlabArgs a{};
    a.channels = C, a.q = p.q, a.inv_n = 1.f / ((float)S * (float)(C / G));
    a.B = B, a.S = S / p.q, a.items = p.items, a.workers = p.workers;
    a.C = C * p.q, a.G = G, a.Cg = C / G, a.Cs = p.Cs, a.Gs = p.Gs, a.slabs = p.slabs, a.TX = p.TX, a.TY = p.TY, a.K = p.K, a.subs = p.subs,
    a.rows = p.rows, a.TYs = p.TYs;
    a.per_row = a.Cg % p.vec == 0 ? a.Cg / p.vec : 1;
    // one number a pack where it lies in one group, else one a group it touches or one a channel
    const int ng = p.groups_of_pack;
    a.width = p.TX * ng;
    a.run = ng == 1 ? a.per_row : (p.q == 1 && ng * a.Cg == p.vec ? 1 : a.Cg);
    a.per_group = a.run * p.q;
    a.by_per_group = make_fastdiv((uint32_t)a.per_group);
    a.by_run = make_fastdiv((uint32_t)a.run);
    auto pow2 = [](int64_t v) { return v > 0 && (v & (v - 1)) == 0; };
    // thread index, from the low bit: packs of a group, groups, rows of a sample, samples
    a.bits = p.q == 1 && pow2(p.TX) && pow2(a.per_row) && p.TX * p.TY == kSlabThreads && a.C % p.Cs == 0 &&
             (ng == 1 ? a.Cg % p.vec == 0 : ng * a.Cg == p.vec);
    const unsigned bits = (unsigned)(a.per_row - 1) | ((unsigned)(p.TYs - 1) * (unsigned)p.TX);
    a.lane_bits = bits & 31u;
    a.warp_bits = bits & ~31u;
    return a;
}

template <typename... Params, typename... Args>
static int launch_clusters(void (*kernel)(Params...), int64_t ctas, int K, size_t smem, cudaStream_t st, Args... args) {
    if (smem > 0) {  // beside up to 36 KB of static shared memory
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return (int)e;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kSlabThreads);
    cfg.dynamicSmemBytes = smem;
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
    // 16-byte packs are always fetched ahead, but for the samples that two CTAs share: those fill the most packs a thread can hold
    constexpr bool can = Held<T, VEC, R>::kAhead, always = can && R < (sizeof(T) == 2 ? 8 : 16);
    const bool ahead = always || p.ahead;
    const size_t smem = ahead ? Held<T, VEC, R>::kStageBytes : 0;
#define SLAB_FWD(NG) (ahead ? k_gn_slab_fwd<T, VEC, R, NG, can> : k_gn_slab_fwd<T, VEC, R, NG, always>)
    auto kernel = SLAB_FWD(1);
    if (VEC > 1 && p.groups_of_pack == 2) kernel = SLAB_FWD((VEC > 1 ? 2 : 1));
    if (VEC > 4 && p.groups_of_pack == 4) kernel = SLAB_FWD((VEC > 4 ? 4 : VEC));
    if (VEC > 2 && p.groups_of_pack == VEC) kernel = SLAB_FWD(VEC);
#undef SLAB_FWD
    return launch_clusters(kernel, ctas, p.K, smem, st, (const T *)x, gamma, beta, a, eps, act, (T *)y, mean, rstd);
}

template <typename T, int VEC, int R>
static int slab_bwd(const SlabPlan &p, const SlabArgs &a, const void *gy, const void *x, const float *gamma, const float *beta, const float *mean,
                    const float *rstd, int act, void *dx, float *part, cudaStream_t st) {
    const int64_t ctas = p.workers * p.slabs * p.K;
    auto kernel = k_gn_slab_bwd<T, VEC, R, 1>;
    if (VEC > 1 && p.groups_of_pack == 2) kernel = k_gn_slab_bwd<T, VEC, R, (VEC > 1 ? 2 : 1)>;
    if (VEC > 4 && p.groups_of_pack == 4) kernel = k_gn_slab_bwd<T, VEC, R, (VEC > 4 ? 4 : VEC)>;
    if (VEC > 2 && p.groups_of_pack == VEC) kernel = k_gn_slab_bwd<T, VEC, R, VEC>;
    return launch_clusters(kernel, ctas, p.K, 0, st, (const T *)gy, (const T *)x, gamma, beta, mean, rstd, a, act, (T *)dx, part);
}

#define SLAB_DISPATCH(FN, MOST, HALF_MOST, ...)                                              \
    do {                                                                               \
        if (type == HGQ_TYPE_F32) {                                                    \
            if (p.vec == 4 && p.R == 1) return FN<float, 4, 1>(__VA_ARGS__);           \
            if (p.vec == 4 && p.R == 4) return FN<float, 4, 4>(__VA_ARGS__);           \
            if (p.vec == 4 && p.R == 8) return FN<float, 4, 8>(__VA_ARGS__);           \
            if (p.vec == 4) return FN<float, 4, MOST>(__VA_ARGS__);                    \
            if (p.vec == 2 && p.R == 1) return FN<float, 2, 1>(__VA_ARGS__);           \
            if (p.vec == 2) return FN<float, 2, 16>(__VA_ARGS__);                      \
            if (p.R == 1) return FN<float, 1, 1>(__VA_ARGS__);                         \
            return FN<float, 1, 16>(__VA_ARGS__);                                      \
        }                                                                              \
        if (type == HGQ_TYPE_BF16) SLAB_HALF(FN, HALF_MOST, __nv_bfloat16, __VA_ARGS__); \
        SLAB_HALF(FN, HALF_MOST, __half, __VA_ARGS__);                                 \
    } while (0)

#define SLAB_HALF(FN, HALF_MOST, T, ...)                                 \
    do {                                                                 \
        if (p.vec == 8 && p.R == 1) return FN<T, 8, 1>(__VA_ARGS__);     \
        if (p.vec == 8 && p.R == 4) return FN<T, 8, 4>(__VA_ARGS__);     \
        if (p.vec == 8) return FN<T, 8, HALF_MOST>(__VA_ARGS__);         \
        if (p.vec == 4 && p.R == 1) return FN<T, 4, 1>(__VA_ARGS__);     \
        if (p.vec == 4 && p.R == 4) return FN<T, 4, 4>(__VA_ARGS__);     \
        if (p.vec == 4) return FN<T, 4, 8>(__VA_ARGS__);                 \
        if (p.vec == 2 && p.R == 1) return FN<T, 2, 1>(__VA_ARGS__);     \
        if (p.vec == 2) return FN<T, 2, 16>(__VA_ARGS__);                \
        if (p.R == 1) return FN<T, 1, 1>(__VA_ARGS__);                   \
        return FN<T, 1, 16>(__VA_ARGS__);                                \
    } while (0)

int gn_slab_fwd(const SlabPlan &p, const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd, int64_t B,
                int64_t S, int C, int G, float eps, int act, int type, cudaStream_t st) {
    const SlabArgs a = slab_args(p, B, S, C, G);
    SLAB_DISPATCH(slab_fwd, 16, 8, p, a, x, gamma, beta, y, mean, rstd, eps, act, st);
}

int gn_slab_bwd(const SlabPlan &p, const void *gy, const void *x, const float *gamma, const float *beta, const float *mean,
                const float *rstd, void *dx, float *part, int64_t B, int64_t S, int C, int G, int act, int type, cudaStream_t st) {
    const SlabArgs a = slab_args(p, B, S, C, G);
    SLAB_DISPATCH(slab_bwd, 8, 4, p, a, gy, x, gamma, beta, mean, rstd, act, dx, part, st);
}

}  // namespace hgq
