// Gated linear recurrence of independent channels,
//     h_t = exp(g_t) h_{t-1} + x_t,   o_t = h_t
// and its gradients: with e_t = exp(g_t) dh_t, what token t hands back to the state before it,
//     dh_t = do_t + e_{t+1},   dx_t = dh_t,   dg_t = e_t h_{t-1},   dh_0 = e_1.
//
// A run of tokens acts on a state as h -> A h + H, with A the product of its decays and H its own final state, and on e in the same form
// from its other end; runs compose.  A warp takes RUN tokens of 32 VEC neighbouring channels, a CTA the runs of a tile of TILE tokens, and walks the
// tiles of its strip of channels: one pass over the data, all sums in fp32, in an order that the sizes alone decide.  Where there are fewer strips than the
// chip has room for, a cluster of CTAs takes neighbouring tiles of a strip at once and exchanges the tiles' (A, H) through shared memory, a barrier for all of them.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/llattn.h"
#include "launch_count.h"

namespace llattn {
namespace rec {

typedef __nv_bfloat16 bf16;
namespace cg = cooperative_groups;
constexpr int WARPS = 8, RUN = 16, TILE = WARPS * RUN, MAX_RANKS = 16;

struct Params {
    const void *x, *g, *d_o;
    const float* h0;          // (B,D) or null: zeros.  Backward: the gradient of the last state, or null
    void *o, *dx, *dg;
    float* h_last;            // (B,D) or null.  Backward: the gradient of the initial state, or null
    float* starts;            // (B,NT,D) or null: the state before every tile
    int T, D, NT, strips;     // strips of channels a sequence
};

template <typename E, int VEC>
struct Row;
template <>
struct Row<bf16, 1> {
    static __device__ __forceinline__ void load(const bf16* p, float (&v)[1]) { v[0] = __bfloat162float(*p); }
    static __device__ __forceinline__ void store(bf16* p, const float (&v)[1]) { *p = __float2bfloat16(v[0]); }
};
template <>
struct Row<bf16, 2> {
    static __device__ __forceinline__ void load(const bf16* p, float (&v)[2]) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
        v[0] = f.x;
        v[1] = f.y;
    }
    static __device__ __forceinline__ void store(bf16* p, const float (&v)[2]) {
        *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v[0], v[1]);
    }
};
template <>
struct Row<float, 1> {
    static __device__ __forceinline__ void load(const float* p, float (&v)[1]) { v[0] = *p; }
    static __device__ __forceinline__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
};
template <>
struct Row<float, 2> {
    static __device__ __forceinline__ void load(const float* p, float (&v)[2]) {
        const float2 f = *reinterpret_cast<const float2*>(p);
        v[0] = f.x;
        v[1] = f.y;
    }
    static __device__ __forceinline__ void store(float* p, const float (&v)[2]) { *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]); }
};

// RUN tokens from t0 on; tokens at or behind `left` and absent channels read as `fill`
template <typename E, int VEC>
__device__ __forceinline__ void load_run(const E* p, long ld, int left, bool there, float fill, float (&v)[RUN][VEC]) {
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
        if (there && i < left) {
            Row<E, VEC>::load(p + i * ld, v[i]);
        } else {
#pragma unroll
            for (int u = 0; u < VEC; ++u) v[i][u] = fill;
        }
    }
}

// A tile's (A, H) to every CTA of the cluster: warp w writes those of ranks w and w + 8.
template <int VEC>
__device__ __forceinline__ void publish(cg::cluster_group& cluster, float2 (*slot)[VEC], int ranks, int warp, int lane, const float (&A)[VEC], const float (&H)[VEC]) {
    for (int x = warp; x < ranks; x += WARPS) {
        float2* to = cluster.map_shared_rank(&slot[lane][0], x);
#pragma unroll
        for (int u = 0; u < VEC; ++u) to[u] = make_float2(A[u], H[u]);
    }
}
// Takes `carry` over the cluster's tiles, in the order of the ranks; `mine` is what reaches this CTA's.
template <int VEC>
__device__ __forceinline__ void over_ranks(const float2 (*all)[32][VEC], int ranks, int rank, int lane, float (&carry)[VEC], float (&mine)[VEC]) {
    for (int x = 0; x < ranks; ++x)
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
            const float2 r = all[x][lane][u];
            if (x == rank) mine[u] = carry[u];
            carry[u] = fmaf(r.x, carry[u], r.y);
        }
}

template <typename X, typename G, int VEC>
__global__ void __launch_bounds__(32 * WARPS, 2) recurrence_fwd_kernel(const __grid_constant__ Params p) {
    chain_wait();
    __shared__ float2 agg[2][WARPS][32][VEC];             // (A, H) of the warps' runs, for every other round
    __shared__ float2 all[2][MAX_RANKS][32][VEC];         // of the cluster's tiles
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank(), unit = blockIdx.x / ranks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = unit / p.strips, c = (unit % p.strips * 32 + lane) * VEC;
    const bool there = c < p.D;
    const long ld = p.D, base = (long)b * p.T * ld + c;
    const X* x = static_cast<const X*>(p.x) + base;
    const G* g = static_cast<const G*>(p.g) + base;
    X* o = static_cast<X*>(p.o) + base;
    if (ranks > 1) cluster.sync();                        // every CTA is there to be written to
    float carry[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u) carry[u] = p.h0 && there ? p.h0[(long)b * p.D + c + u] : 0.f;
    int par = 0;
    for (int first = 0; first < p.NT; first += ranks, par ^= 1) {
        const int tile = first + rank, t0 = tile * TILE + warp * RUN, left = p.T - t0;      // (a tile behind the last changes nothing)
        float v[RUN][VEC], a[RUN][VEC];
        load_run<X, VEC>(x + (long)t0 * ld, ld, left, there, 0.f, v);
        load_run<G, VEC>(g + (long)t0 * ld, ld, left, there, 0.f, a);
        float A[VEC], H[VEC], h[VEC], mine[VEC];
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
            A[u] = 1.f;
            H[u] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < RUN; ++i)
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
                a[i][u] = expf(a[i][u]);
                A[u] *= a[i][u];
                H[u] = fmaf(a[i][u], H[u], v[i][u]);
            }
#pragma unroll
        for (int u = 0; u < VEC; ++u) agg[par][warp][lane][u] = make_float2(A[u], H[u]);
        __syncthreads();
        if (ranks == 1) {
#pragma unroll
            for (int u = 0; u < VEC; ++u) mine[u] = carry[u];
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
#pragma unroll
                for (int u = 0; u < VEC; ++u) {
                    const float2 r = agg[par][w][lane][u];
                    if (w == warp) h[u] = carry[u];
                    carry[u] = fmaf(r.x, carry[u], r.y);
                }
        } else {
            float Ab[VEC], Hb[VEC];                       // of the runs before this warp's; then of the tile
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
                A[u] = 1.f;
                H[u] = 0.f;
            }
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
#pragma unroll
                for (int u = 0; u < VEC; ++u) {
                    const float2 r = agg[par][w][lane][u];
                    if (w == warp) {
                        Ab[u] = A[u];
                        Hb[u] = H[u];
                    }
                    A[u] *= r.x;
                    H[u] = fmaf(r.x, H[u], r.y);
                }
            publish<VEC>(cluster, all[par][rank], ranks, warp, lane, A, H);
            cluster.sync();
            over_ranks<VEC>(all[par], ranks, rank, lane, carry, mine);
#pragma unroll
            for (int u = 0; u < VEC; ++u) h[u] = fmaf(Ab[u], mine[u], Hb[u]);
        }
        if (p.starts && warp == 0 && there && tile < p.NT) Row<float, VEC>::store(p.starts + ((long)b * p.NT + tile) * p.D + c, mine);
        if (there) {
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                if (i < left) {
#pragma unroll
                    for (int u = 0; u < VEC; ++u) h[u] = fmaf(a[i][u], h[u], v[i][u]);
                    Row<X, VEC>::store(o + (long)(t0 + i) * ld, h);
                }
            }
        }
    }
    if (p.h_last && rank == 0 && warp == 0 && there) Row<float, VEC>::store(p.h_last + (long)b * p.D + c, carry);
}

// The same from the other end: e takes the place of the state, the cluster's tiles are counted from the last one.
template <typename X, typename G, int VEC>
__global__ void __launch_bounds__(32 * WARPS, 2) recurrence_bwd_kernel(const __grid_constant__ Params p) {
    chain_wait();
    __shared__ float agg[2][3][WARPS][32][VEC];           // A, H and E of the warps' runs
    __shared__ float2 all[2][MAX_RANKS][32][VEC];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank(), unit = blockIdx.x / ranks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = unit / p.strips, c = (unit % p.strips * 32 + lane) * VEC;
    const bool there = c < p.D;
    const long ld = p.D, base = (long)b * p.T * ld + c;
    const X* x = static_cast<const X*>(p.x) + base;
    const G* g = static_cast<const G*>(p.g) + base;
    const X* d_o = static_cast<const X*>(p.d_o) + base;
    X* dx = static_cast<X*>(p.dx) + base;
    G* dg = static_cast<G*>(p.dg) + base;
    if (ranks > 1) cluster.sync();
    float carry[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u) carry[u] = p.h0 && there ? p.h0[(long)b * p.D + c + u] : 0.f;
    int par = 0;
    for (int first = p.NT - 1; first >= 0; first -= ranks, par ^= 1) {
        const int tile = first - rank, t0 = tile * TILE + warp * RUN, left = tile < 0 ? 0 : p.T - t0;
        float v[RUN][VEC], a[RUN][VEC], d[RUN][VEC];
        load_run<X, VEC>(x + (long)t0 * ld, ld, left, there, 0.f, v);
        load_run<G, VEC>(g + (long)t0 * ld, ld, left, there, 0.f, a);
        load_run<X, VEC>(d_o + (long)t0 * ld, ld, left, there, 0.f, d);
        float A[VEC], H[VEC], E[VEC], h[VEC], e[VEC], mine[VEC];
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
            A[u] = 1.f;
            H[u] = E[u] = 0.f;
            h[u] = there && tile >= 0 ? p.starts[((long)b * p.NT + tile) * p.D + c + u] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < RUN; ++i)
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
                a[i][u] = expf(a[i][u]);
                A[u] *= a[i][u];
                H[u] = fmaf(a[i][u], H[u], v[i][u]);
            }
#pragma unroll
        for (int i = RUN - 1; i >= 0; --i)
#pragma unroll
            for (int u = 0; u < VEC; ++u) E[u] = a[i][u] * (d[i][u] + E[u]);
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
            agg[par][0][warp][lane][u] = A[u];
            agg[par][1][warp][lane][u] = H[u];
            agg[par][2][warp][lane][u] = E[u];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < VEC; ++u)
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
                if (w < warp) h[u] = fmaf(agg[par][0][w][lane][u], h[u], agg[par][1][w][lane][u]);
        if (ranks == 1) {
#pragma unroll
            for (int u = 0; u < VEC; ++u)
#pragma unroll
                for (int w = WARPS - 1; w >= 0; --w) {
                    if (w == warp) e[u] = carry[u];
                    carry[u] = fmaf(agg[par][0][w][lane][u], carry[u], agg[par][2][w][lane][u]);
                }
        } else {
            float Ab[VEC], Eb[VEC];                       // of the runs behind this warp's; then of the tile
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
                A[u] = 1.f;
                E[u] = 0.f;
#pragma unroll
                for (int w = WARPS - 1; w >= 0; --w) {
                    const float aw = agg[par][0][w][lane][u];
                    if (w == warp) {
                        Ab[u] = A[u];
                        Eb[u] = E[u];
                    }
                    A[u] *= aw;
                    E[u] = fmaf(aw, E[u], agg[par][2][w][lane][u]);
                }
            }
            publish<VEC>(cluster, all[par][rank], ranks, warp, lane, A, E);
            cluster.sync();
            over_ranks<VEC>(all[par], ranks, rank, lane, carry, mine);
#pragma unroll
            for (int u = 0; u < VEC; ++u) e[u] = fmaf(Ab[u], mine[u], Eb[u]);
        }
        // the states before the run's tokens, in the place of x
#pragma unroll
        for (int i = 0; i < RUN; ++i)
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
                const float next = fmaf(a[i][u], h[u], v[i][u]);
                v[i][u] = h[u];
                h[u] = next;
            }
        if (there) {
#pragma unroll
            for (int i = RUN - 1; i >= 0; --i) {
                if (i < left) {
                    float dh[VEC], dgi[VEC];
#pragma unroll
                    for (int u = 0; u < VEC; ++u) {
                        dh[u] = d[i][u] + e[u];
                        e[u] = a[i][u] * dh[u];
                        dgi[u] = e[u] * v[i][u];
                    }
                    Row<X, VEC>::store(dx + (long)(t0 + i) * ld, dh);
                    Row<G, VEC>::store(dg + (long)(t0 + i) * ld, dgi);
                }
            }
        }
    }
    if (p.h_last && rank == 0 && warp == 0 && there) Row<float, VEC>::store(p.h_last + (long)b * p.D + c, carry);
}

template <typename X, typename G>
__global__ void __launch_bounds__(256) recurrence_step_kernel(float* h, const X* x, const G* g, X* o, long n) {
    chain_wait();
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v[1], a[1];
    Row<X, 1>::load(x + i, v);
    Row<G, 1>::load(g + i, a);
    v[0] = fmaf(expf(a[0]), h[i], v[0]);
    h[i] = v[0];
    Row<X, 1>::store(o + i, v);
}

// Clusters of as many CTAs as fill the chip twice over, and no more than there are tiles.
inline int ranks_of(long units, int NT) {
    int n = 1;
    while (n < MAX_RANKS && 2 * n <= NT && units * n < 2 * 148) n *= 2;
    return n;
}
template <typename KernT>
cudaError_t launch(KernT kern, const Params& p, long units, cudaStream_t st) {
    const int n = ranks_of(units, p.NT);
    if (n > 8) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = n;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * n));
    cfg.blockDim = dim3(32 * WARPS);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return e;
}
template <typename X, typename G>
cudaError_t scan(bool backward, Params p, int B, cudaStream_t st) {
    const bool pairs = p.D % 2 == 0;
    p.strips = (p.D + (pairs ? 64 : 32) - 1) / (pairs ? 64 : 32);
    const long units = (long)B * p.strips;
    if (backward) return pairs ? launch(recurrence_bwd_kernel<X, G, 2>, p, units, st) : launch(recurrence_bwd_kernel<X, G, 1>, p, units, st);
    return pairs ? launch(recurrence_fwd_kernel<X, G, 2>, p, units, st) : launch(recurrence_fwd_kernel<X, G, 1>, p, units, st);
}
int scan_of(bool backward, int x_f32, int g_f32, const Params& p, int B, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (x_f32) e = scan<float, float>(backward, p, B, st);
    else if (g_f32) e = scan<bf16, float>(backward, p, B, st);
    else e = scan<bf16, bf16>(backward, p, B, st);
    return (int)e;
}
int check(int x_f32, int g_f32, long B, long T, long D) {
    if (B < 1 || T < 1 || D < 1 || (x_f32 && !g_f32)) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    if (T > (1 << 30) || B * ((D + 31) / 32) > 0x7fffffffl) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    return 0;
}

}  // namespace rec
}  // namespace llattn

using namespace llattn;

extern "C" {

size_t llattn_recurrence_states_bytes(int B, int T, int D) {
    if (rec::check(0, 0, B, T, D) != 0) return 0;
    return (size_t)B * ((T + rec::TILE - 1) / rec::TILE) * D * sizeof(float);
}

int llattn_recurrence_fwd(const void* x, int x_is_f32, const void* g, int g_is_f32, const float* h0, void* o, float* h_last, float* states,
                          int B, int T, int D, void* stream) {
    const int rc = rec::check(x_is_f32, g_is_f32, B, T, D);
    if (rc != 0) return rc;
    if (!x || !g || !o) return LLATTN_ERR_NULL;
    if (misaligned(16, {x, g, h0, o, h_last, states})) return LLATTN_ERR_ALIGNMENT;
    rec::Params p = {};
    p.x = x;
    p.g = g;
    p.h0 = h0;
    p.o = o;
    p.h_last = h_last;
    p.starts = states;
    p.T = T;
    p.D = D;
    p.NT = (T + rec::TILE - 1) / rec::TILE;
    return rec::scan_of(false, x_is_f32, g_is_f32, p, B, stream);
}

int llattn_recurrence_bwd(const void* x, int x_is_f32, const void* g, int g_is_f32, const float* states, const void* d_o, const float* dh_last,
                          void* dx, void* dg, float* dh0, int B, int T, int D, void* stream) {
    const int rc = rec::check(x_is_f32, g_is_f32, B, T, D);
    if (rc != 0) return rc;
    if (!x || !g || !states || !d_o || !dx || !dg) return LLATTN_ERR_NULL;
    if (misaligned(16, {x, g, states, d_o, dh_last, dx, dg, dh0})) return LLATTN_ERR_ALIGNMENT;
    rec::Params p = {};
    p.x = x;
    p.g = g;
    p.d_o = d_o;
    p.h0 = dh_last;
    p.dx = dx;
    p.dg = dg;
    p.h_last = dh0;
    p.starts = const_cast<float*>(states);
    p.T = T;
    p.D = D;
    p.NT = (T + rec::TILE - 1) / rec::TILE;
    return rec::scan_of(true, x_is_f32, g_is_f32, p, B, stream);
}

int llattn_recurrence_step(float* h, const void* x, int x_is_f32, const void* g, int g_is_f32, void* o, int B, int D, void* stream) {
    const int rc = rec::check(x_is_f32, g_is_f32, B, 1, D);
    if (rc != 0) return rc;
    if (!h || !x || !g || !o) return LLATTN_ERR_NULL;
    if (misaligned(16, {h, x, g, o})) return LLATTN_ERR_ALIGNMENT;
    const long n = (long)B * D;
    if ((n + 255) / 256 > 0x7fffffffl) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    const unsigned grid = (unsigned)((n + 255) / 256);
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    typedef rec::bf16 bf16;
    if (x_is_f32)
        e = launch_chained(rec::recurrence_step_kernel<float, float>, grid, 256, 0, st, h, (const float*)x, (const float*)g, (float*)o, n);
    else if (g_is_f32)
        e = launch_chained(rec::recurrence_step_kernel<bf16, float>, grid, 256, 0, st, h, (const bf16*)x, (const float*)g, (bf16*)o, n);
    else
        e = launch_chained(rec::recurrence_step_kernel<bf16, bf16>, grid, 256, 0, st, h, (const bf16*)x, (const bf16*)g, (bf16*)o, n);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return (int)e;
}

}  // extern "C"
