// One decoding step of the sliding-window attention: the token's k and v go into their slot, its R = H / G queries a group attend to the slots that hold tokens.
//
// It is bound by the cache, each held slot read once: 4 K bytes and 4 K R flops a slot and group, more than fp32 units do beside 6.4 TB/s from four heads a
// group on; so the products are warp-level matrix instructions, with slots as the long side and heads as the short one (eight heads fill a tile),
//     S^T (16 slots x 8 heads) = K Q^T,   O^T (K columns x 8 heads) += V^T P^T.
// Operands go from memory to the registers that the instructions read, 16 bytes a load: the order of a product's reduction index is free, so a lane takes 8
// neighbouring columns of k as the indices of two instructions, and 8 neighbouring columns of v as the rows of eight.  No shared memory, no barrier in the loop.
// P is multiplied in two bf16 terms, exact to 2^-16: one term, 2^-8, left outputs 2.3e-3 off 64 bits, of which 1.7e-3 are their own rounding.  The second instruction costs
// 2 % of the figures below, 1 to 4 % of other calls.
//
// The slots of a (sequence, group) are spread over the warps of a cluster of CTAs, which write their maxima, sums and outputs to the shared memory of the one that joins them:
// one launch, no workspace, the order of every sum given by the sizes.
// 64 sequences, 32 heads on 8, K = 128, 2052 slots: 93 us, 5.8 TB/s.  One sequence, 4100 slots: 8.8 us, latency (count, slots,
// a cluster's barrier and two joins one after another).
#include <cooperative_groups.h>

#include "../../include/llattn.h"
#include "llattn_testing.h"
#include "window.cuh"

namespace llattn {
namespace win {

namespace step {
namespace cg = cooperative_groups;
constexpr int BLOCK = 16;                      // slots a warp takes at once
constexpr int MAX_RANKS = 16;
template <int NT>
struct Cta {
    static constexpr int WARPS = NT == 1 ? 8 : 4;      // (16 heads: twice the registers, twice the shared memory a warp)
};

struct Params {
    const bf16 *q, *k, *v;
    bf16 *kc, *vc, *o;
    long long* counts;
    int H, G, R, window, sinks;
    float scale;
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {       // of an 8 x 8 matrix, a row four lanes
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 slot_words(const bf16* p, bool there) {
    return there ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}
// NT tiles of eight heads from h0 on, q at the first of them
template <int K, int NT>
__device__ __forceinline__ void load_queries(uint32_t (&qf)[NT][K / 8], const Params& p, const bf16* q, int h0, int r, int c) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < K / 32; ++i) {
            const uint4 w = slot_words(q + (long)(8 * n + r) * K + (c + 4 * i) * 8, h0 + 8 * n + r < p.R);
            qf[n][4 * i] = w.x;
            qf[n][4 * i + 1] = w.y;
            qf[n][4 * i + 2] = w.z;
            qf[n][4 * i + 3] = w.w;
        }
}
// the cluster's barrier in two halves; what is written before one is there behind the other
__device__ __forceinline__ void arrive(const cg::cluster_group&) { cg::cluster_group::barrier_arrive(); }
__device__ __forceinline__ void wait(const cg::cluster_group&) { cg::cluster_group::barrier_wait(); }
}  // namespace step

// NT tiles of eight heads together
template <int K, int NT>
__global__ void __launch_bounds__(32 * step::Cta<NT>::WARPS, 2) window_step_kernel(const __grid_constant__ step::Params p) {
    chain_wait();
    using namespace step;
    constexpr int HEADS = 8 * NT, WARPS = Cta<NT>::WARPS;
    __shared__ float sO[WARPS][HEADS][K + 4];            // (the warps' outputs; the CTA's in the first)
    __shared__ float sM[WARPS][HEADS], sL[WARPS][HEADS];
    // what the cluster's CTAs send this one: their outputs, maxima and sums of the elements (head, column) that it joins
    __shared__ float rO[HEADS * K], rM[MAX_RANKS][HEADS], rL[MAX_RANKS][HEADS];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
    const int unit = blockIdx.x / ranks, grp = unit % p.G;
    const long b = unit / p.G;
    const int slots = p.sinks + p.window, stride = ranks * WARPS * BLOCK, first = (rank * WARPS + warp) * BLOCK;
    const long ld = (long)p.G * K;
    bf16 *kb = p.kc + (b * slots * p.G + grp) * K, *vb = p.vc + (b * slots * p.G + grp) * K;
    // what does not depend on the count is on its way before the count is there
    arrive(cluster);
    const long long count = p.counts[unit];
    const uint4 none = make_uint4(0, 0, 0, 0);
    const uint4 new_k = lane < K / 8 ? reinterpret_cast<const uint4*>(p.k + (long)unit * K)[lane] : none;
    const uint4 new_v = lane < K / 8 ? reinterpret_cast<const uint4*>(p.v + (long)unit * K)[lane] : none;
    uint32_t qf[NT][K / 8];
    load_queries<K, NT>(qf, p, p.q + (b * p.H + grp * p.R) * K, 0, r, c);
    const long long seen = count > 0 ? count : 0;
    const int slot = (int)(seen < p.sinks ? seen : p.sinks + (seen - p.sinks) % p.window), held = (int)min((long long)slots, seen + 1);
    // the warp whose block of slots the new token falls into stores it, and reads it back with the others
    if (slot / BLOCK % (ranks * WARPS) == rank * WARPS + warp) {
        if (lane < K / 8) {
            reinterpret_cast<uint4*>(kb + slot * ld)[lane] = new_k;
            reinterpret_cast<uint4*>(vb + slot * ld)[lane] = new_v;
        }
        __syncwarp();
    }
    const float scale = p.scale * LOG2E;
    for (int h0 = 0; h0 < p.R; h0 += HEADS) {
        if (h0 > 0) {
            load_queries<K, NT>(qf, p, p.q + (b * p.H + grp * p.R + h0) * K, h0, r, c);
        }
        float acc[NT][K / 16][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < K / 16; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
        }
        for (int s0 = first; s0 < held; s0 += stride) {
            uint4 kw[2][K / 32], vw[K / 64][4];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < K / 32; ++i) kw[u][i] = slot_words(kb + (s0 + r + 8 * u) * ld + (c + 4 * i) * 8, s0 + r + 8 * u < held);
#pragma unroll
            for (int i = 0; i < K / 64; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int s = s0 + 2 * c + (u & 1) + 8 * (u >> 1);
                    vw[i][u] = slot_words(vb + s * ld + 64 * i + 8 * r, s < held);
                }
            uint32_t pf[NT][2], pl[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < K / 32; ++i) {
                    mma(d, kw[0][i].x, kw[1][i].x, kw[0][i].y, kw[1][i].y, qf[n][4 * i], qf[n][4 * i + 1]);
                    mma(d, kw[0][i].z, kw[1][i].z, kw[0][i].w, kw[1][i].w, qf[n][4 * i + 2], qf[n][4 * i + 3]);
                }
                // slots r and r + 8 of heads 2 c and 2 c + 1
                const bool in0 = s0 + r < held, in1 = s0 + r + 8 < held;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float y0 = in0 ? d[u] * scale : -INFINITY, y1 = in1 ? d[2 + u] * scale : -INFINITY;
                    float top = fmaxf(y0, y1);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    top = fmaxf(top, m[n][u]);
                    const float ref = top == -INFINITY ? 0.f : top;
                    const float f = exp2_fast(m[n][u] - ref);
                    m[n][u] = top;
                    d[u] = exp2_fast(y0 - ref);
                    d[2 + u] = exp2_fast(y1 - ref);
                    l[n][u] = fmaf(l[n][u], f, d[u] + d[2 + u]);
#pragma unroll
                    for (int i = 0; i < K / 16; ++i) {
                        acc[n][i][u] *= f;
                        acc[n][i][2 + u] *= f;
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    pf[n][u] = transposed(cut_bf16(d[2 * u], d[2 * u + 1]));
                    pl[n][u] = transposed(pack_bf16(cut_off(d[2 * u]), cut_off(d[2 * u + 1])));
                }
            }
            // rows of a tile: columns 64 i + 8 r + 2 t (d0, d1) and the one behind it (d2, d3)
#pragma unroll
            for (int i = 0; i < K / 64; ++i)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t w0 = t == 0 ? vw[i][0].x : t == 1 ? vw[i][0].y : t == 2 ? vw[i][0].z : vw[i][0].w;
                    const uint32_t w1 = t == 0 ? vw[i][1].x : t == 1 ? vw[i][1].y : t == 2 ? vw[i][1].z : vw[i][1].w;
                    const uint32_t w2 = t == 0 ? vw[i][2].x : t == 1 ? vw[i][2].y : t == 2 ? vw[i][2].z : vw[i][2].w;
                    const uint32_t w3 = t == 0 ? vw[i][3].x : t == 1 ? vw[i][3].y : t == 2 ? vw[i][3].z : vw[i][3].w;
                    const uint32_t a0 = __byte_perm(w0, w1, 0x5410), a1 = __byte_perm(w0, w1, 0x7632), a2 = __byte_perm(w2, w3, 0x5410), a3 = __byte_perm(w2, w3, 0x7632);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma(acc[n][4 * i + t], a0, a1, a2, a3, pf[n][0], pf[n][1]);
                        mma(acc[n][4 * i + t], a0, a1, a2, a3, pl[n][0], pl[n][1]);
                    }
                }
        }
        // the warps' parts, joined in the CTA, then in the cluster
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int h = 8 * n + 2 * c + u;
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][u] += __shfl_xor_sync(0xffffffffu, l[n][u], x);
                if (r == 0) {
                    sM[warp][h] = m[n][u];
                    sL[warp][h] = l[n][u];
                }
#pragma unroll
                for (int i = 0; i < K / 16; ++i) {
                    const int col = 64 * (i >> 2) + 8 * r + 2 * (i & 3);
                    *reinterpret_cast<float2*>(&sO[warp][h][col]) = make_float2(acc[n][i][u], acc[n][i][2 + u]);
                }
            }
        __syncthreads();
        // the cluster's CTAs have begun, and read what they were sent before
        wait(cluster);
        const int each = HEADS * K / ranks;
        for (int e = threadIdx.x; e < HEADS * K; e += 32 * WARPS) {
            const int h = e / K, col = e % K, to = e / each;
            float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sM[w][h]);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = exp2_fast(sM[w][h] - ref);
                sum = fmaf(f, sL[w][h], sum);
                o = fmaf(f, sO[w][h][col], o);
            }
            *cluster.map_shared_rank(&rO[rank * each + e - to * each], to) = o;
            if (e == to * each || col == 0) {
                *cluster.map_shared_rank(&rM[rank][h], to) = top;
                *cluster.map_shared_rank(&rL[rank][h], to) = sum;
            }
        }
        arrive(cluster);
        wait(cluster);
        for (int i = threadIdx.x; i < each; i += 32 * WARPS) {
            const int e = rank * each + i, h = e / K, col = e % K;
            float top = -INFINITY, sum = 0.f, o = 0.f;
            for (int x = 0; x < ranks; ++x) top = fmaxf(top, rM[x][h]);
#pragma unroll 4
            for (int x = 0; x < ranks; ++x) {
                const float f = exp2_fast(rM[x][h] - top);
                sum = fmaf(f, rL[x][h], sum);
                o = fmaf(f, rO[x * each + i], o);
            }
            if (h0 + h < p.R) p.o[(b * p.H + grp * p.R + h0 + h) * K + col] = __float2bfloat16(o / sum);
        }
        if (h0 + HEADS < p.R) arrive(cluster);
    }
    // every CTA of the cluster has read the count
    if (rank == 0 && threadIdx.x == 0) p.counts[unit] = seen + 1;
}

constexpr int PORTABLE_RANKS = 8;                // what every device places
// Clusters of 1 to 16 CTAs, of at most `most`: as many as leave every warp two blocks of slots, up to two CTAs an SM.
static int ranks_of(long units, int slots, int warps, int most) {
    int n = 1;
    while (2 * n <= most && slots > n * warps * step::BLOCK * 2 && units * n < 148) n *= 2;
    return n;
}
template <int K, int NT>
static cudaError_t launch_step(const step::Params& p, long units, cudaStream_t st) {
    const auto kern = window_step_kernel<K, NT>;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(32 * step::Cta<NT>::WARPS);
    cfg.stream = st;
    cfg.attrs = attr;
    const auto clusters_of = [&](int n) {
        attr[0].val.clusterDim.x = n;
        cfg.gridDim = dim3((unsigned)(units * n));
    };
    int n = ranks_of(units, p.sinks + p.window, step::Cta<NT>::WARPS, step::MAX_RANKS);
    cudaError_t e;
    if (n > PORTABLE_RANKS) {
        static thread_local int asked = -1, most = 0;     // the device that was asked for clusters of 16, and the largest that it places
        int dev;
        e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (asked != dev) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            clusters_of(n);
            cfg.numAttrs = 1;
            int places = 0;
            e = cudaOccupancyMaxActiveClusters(&places, kern, &cfg);
            if (e != cudaSuccess) return e;
            most = places > 0 ? step::MAX_RANKS : PORTABLE_RANKS;
            asked = dev;
        }
        n = ranks_of(units, p.sinks + p.window, step::Cta<NT>::WARPS, most);
    }
    clusters_of(n);
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return e;
}

cudaError_t decode_step(const bf16* q, const bf16* k, const bf16* v, bf16* kc, bf16* vc, long long* counts, bf16* o, int B, int H, int G, int K, int window,
                        int sinks, float scale, cudaStream_t st) {
    const step::Params p = {q, k, v, kc, vc, o, counts, H, G, H / G, window, sinks, scale};
    const long units = (long)B * G;
    if (p.R <= 8) return K == 64 ? launch_step<64, 1>(p, units, st) : launch_step<128, 1>(p, units, st);
    return K == 64 ? launch_step<64, 2>(p, units, st) : launch_step<128, 2>(p, units, st);
}

}  // namespace win
}  // namespace llattn

extern "C" int llattn_testing_window_step_ranks(long units, int slots, int heads, int most) {
    using namespace llattn::win;
    return ranks_of(units, slots, heads <= 8 ? step::Cta<1>::WARPS : step::Cta<2>::WARPS, most);
}
