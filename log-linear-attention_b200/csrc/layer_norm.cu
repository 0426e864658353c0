// Layer norm over rows of N values and its gradients:
//     y  = (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//     dx = rstd (z - mean(z) - xhat mean(z xhat)),   z = w dy,  xhat = (x - mean) rstd
//     dw = sum over rows of dy xhat,   db = sum over rows of dy
// w absent is ones, b absent zeros.  All sums in fp32; the variance from the differences to the mean.
//
// Bound by memory as long as few instructions are issued a value.  CTAs stay on the chip and take rows in turn, LANES lanes a row, which comes two or three rows ahead of
// its sums by asynchronous copies to shared memory, each lane its own 16-byte words (single values where rows do not start at their boundaries).  A lane sees the same
// columns of every row: w and b stay in its registers (re-read from L1 for every row they cost bf16 rows more than the rows themselves, 61 us for 32768 x 2048), and dw
// and db are sums in registers, then over the CTA's rows in shared memory, then over the CTAs in a second kernel, always in the same order.  Arithmetic is
// on pairs (f32x2).  Rows longer than a CTA's registers hold are read again for each sum, and the column sums are a pass of their own.
// 32768 x 2048 bf16: forward 51 us, backward with dw and db 80 us, 5.3 and 5.0 TB/s.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/llattn.h"
#include "launch_count.h"
#include "pairs.cuh"

namespace llattn {
namespace norm {

typedef __nv_bfloat16 bf16;

struct Params {
    const void *x, *w, *b, *dy;
    void *y, *dx, *dw, *db;
    float *mean, *rstd;       // a row each
    float* part;              // (parts, 2, N): partial dw and db
    long rows;
    int N, parts;
    float eps;
};

__device__ __forceinline__ float get(const float* p) { return *p; }
__device__ __forceinline__ float get(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16* p, float v) { *p = __float2bfloat16(v); }

// VEC neighbouring values of a row as N numbers; VEC is 1 or a multiple of a 16-byte word
template <int VEC>
struct Lane {
    typedef F2 T;
    static constexpr int N = VEC / 2;
    static __device__ __forceinline__ void load(const float* p, T (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float4 f = *reinterpret_cast<const float4*>(p + 2 * i);
            v[i] = pair(f.x, f.y);
            v[i + 1] = pair(f.z, f.w);
        }
    }
    static __device__ __forceinline__ void load(const bf16* p, T (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 q = *reinterpret_cast<const uint4*>(p + 2 * i);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i + k] = pair(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
        }
    }
    static __device__ __forceinline__ void store(float* p, const T (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 a = both(v[i]), b = both(v[i + 1]);
            *reinterpret_cast<float4*>(p + 2 * i) = make_float4(a.x, a.y, b.x, b.y);
        }
    }
    static __device__ __forceinline__ void store(bf16* p, const T (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = both(v[i + k]);
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(f.y), "f"(f.x));
            }
            *reinterpret_cast<uint4*>(p + 2 * i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};
template <>
struct Lane<1> {
    typedef float T;
    static constexpr int N = 1;
    template <typename E>
    static __device__ __forceinline__ void load(const E* p, T (&v)[1]) { v[0] = get(p); }
    template <typename E>
    static __device__ __forceinline__ void store(E* p, const T (&v)[1]) { put(p, v[0]); }
};

// Sum over the LANES lanes of a row: a warp's or fewer by exchange, more through shared memory (all threads of the CTA take part).
template <int LANES, int THREADS, int V>
__device__ __forceinline__ void row_sum(float (&s)[V], float (*sh)[THREADS / 32]) {
#pragma unroll
    for (int d = (LANES < 32 ? LANES : 32) / 2; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
    if constexpr (LANES > 32) {
        constexpr int W = LANES / 32;
        const int warp = threadIdx.x >> 5, first = warp / W * W;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < V; ++i) sh[i][warp] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s[i] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) s[i] += sh[i][first + w];
        }
    }
}

// The rows to come, in shared memory.  Words of 16 bytes, or of one fp32 value: [STAGES][ITER][TENSORS][THREADS], each lane's own.  bf16 rows that do not start
// at 16-byte boundaries: [STAGES][TENSORS][GROUPS] rows as they are in memory, from the 4-byte boundary at or before their start on (there are no copies
// of two bytes), so that a lane's values come with another lane's copies.
template <typename X, int VEC, int ITER, int LANES, int THREADS, int TENSORS>
struct Ring {
    static constexpr bool SHARED = VEC * sizeof(X) == 2;
    static constexpr int GROUPS = THREADS / LANES, CAP = LANES * ITER * VEC + (SHARED ? 8 : 0);         // values of a row
    static constexpr int BYTES = VEC * ITER * (int)sizeof(X), STAGES = BYTES * TENSORS > 64 ? 3 : 4;
    static constexpr size_t SIZE = (size_t)STAGES * TENSORS * GROUPS * CAP * sizeof(X);
    static __device__ __forceinline__ X* word(X* ring, int stage, int i, int t) {
        return ring + (((stage * ITER + i) * TENSORS + t) * THREADS + (int)threadIdx.x) * VEC;
    }
    static __device__ __forceinline__ X* whole(X* ring, int stage, int t) {
        return ring + ((stage * TENSORS + t) * GROUPS + (int)threadIdx.x / LANES) * CAP;
    }
    static __device__ __forceinline__ void bring(X* ring, int stage, int t, const X* x, long row, long rows, int N, int lane) {
        if constexpr (SHARED) {
            const int odd = (int)(row * N & 1), words = (N + odd + 1) / 2;
            const X* from = x + row * N - odd;
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(whole(ring, stage, t));
            const bool last = row + 1 == rows && (N + odd) % 2 != 0;                 // the tensor ends in the middle of the last word
#pragma unroll
            for (int i = 0; i < ITER / 2 + 1; ++i) {
                const int k = i * LANES + lane;
                if (k < words)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(to + 4 * k), "l"(from + 2 * k), "r"(last && k + 1 == words ? 2 : 4) : "memory");
            }
        } else {
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                const int c = (i * LANES + lane) * VEC;
                const uint32_t to = (uint32_t)__cvta_generic_to_shared(word(ring, stage, i, t));
                if (c < N) {
                    if constexpr (VEC * sizeof(X) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(x + row * N + c) : "memory");
                    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to), "l"(x + row * N + c) : "memory");
                }
            }
        }
    }
    template <typename T, int N_>
    static __device__ __forceinline__ void read(X* ring, int stage, int i, int t, long row, int N, int lane, T (&v)[N_]) {
        if constexpr (SHARED) Lane<VEC>::load(whole(ring, stage, t) + (int)(row * N & 1) + i * LANES + lane, v);
        else Lane<VEC>::load(word(ring, stage, i, t), v);
    }
};
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

// CTA i of the grid takes the rows from i GROUPS on, GROUPS = THREADS / LANES of them at once, then those a grid further on.
template <typename X, typename W, int VEC, int ITER, int LANES, int THREADS>
__global__ void __launch_bounds__(THREADS, 2) layer_norm_fwd_kernel(const __grid_constant__ Params p) {
    chain_wait();
    constexpr int GROUPS = THREADS / LANES;
    using R = Ring<X, VEC, ITER, LANES, THREADS, 1>;
    using L = Lane<VEC>;
    typedef typename L::T T;
    __shared__ float sh[2][1][THREADS / 32];
    extern __shared__ __align__(16) unsigned char ring_raw[];
    X* ring = reinterpret_cast<X*>(ring_raw);
    const int N = p.N, lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.f / (float)N;
    const X* x = static_cast<const X*>(p.x);
    const W *w = static_cast<const W*>(p.w), *b = static_cast<const W*>(p.b);
    const long stride = (long)gridDim.x * GROUPS, first = (long)blockIdx.x * GROUPS + group;
    const auto fetch = [&](long row, int stage) {
        if (row < p.rows) R::bring(ring, stage, 0, x, row, p.rows, N, lane);
        copies_commit();
    };
#pragma unroll
    for (int k = 0; k < R::STAGES - 1; ++k) fetch(first + k * stride, k);
    T wv[ITER][L::N], bv[ITER][L::N];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * LANES + lane) * VEC;
#pragma unroll
        for (int u = 0; u < L::N; ++u) {
            wv[i][u] = splat<T>(1.f);
            bv[i][u] = splat<T>(0.f);
        }
        if (w && c < N) L::load(w + c, wv[i]);
        if (b && c < N) L::load(b + c, bv[i]);
    }
    int stage = 0;
    for (long row = first; row - group < p.rows; row += stride, stage = stage + 1 == R::STAGES ? 0 : stage + 1) {
        copies_but<R::STAGES - 2>();
        if constexpr (R::SHARED) __syncthreads();
        T v[ITER][L::N], t = splat<T>(0.f);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (row < p.rows && (i * LANES + lane) * VEC < N) {
                R::read(ring, stage, i, 0, row, N, lane, v[i]);
            } else {
#pragma unroll
                for (int u = 0; u < L::N; ++u) v[i][u] = splat<T>(0.f);
            }
#pragma unroll
            for (int u = 0; u < L::N; ++u) t = add(t, v[i][u]);
        }
        fetch(row + (R::STAGES - 1) * stride, stage == 0 ? R::STAGES - 1 : stage - 1);       // (where the row before this one was)
        float s[1] = {total(t)}, ss[1];
        row_sum<LANES, THREADS>(s, sh[0]);
        const float mean = s[0] * inv;
        t = splat<T>(0.f);
#pragma unroll
        for (int i = 0; i < ITER; ++i)
            if ((i * LANES + lane) * VEC < N)
#pragma unroll
                for (int u = 0; u < L::N; ++u) {
                    v[i][u] = add(v[i][u], splat<T>(-mean));
                    t = fma2(v[i][u], v[i][u], t);
                }
        ss[0] = total(t);
        row_sum<LANES, THREADS>(ss, sh[1]);
        const float rstd = rsqrtf(ss[0] * inv + p.eps);
        if (row < p.rows) {
            X* y = static_cast<X*>(p.y) + row * N;
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                const int c = (i * LANES + lane) * VEC;
                if (c < N) {
#pragma unroll
                    for (int u = 0; u < L::N; ++u) v[i][u] = fma2(mul(v[i][u], splat<T>(rstd)), wv[i][u], bv[i][u]);
                    L::store(y + c, v[i]);
                }
            }
            if (lane == 0 && p.mean) {
                p.mean[row] = mean;
                p.rstd[row] = rstd;
            }
        }
    }
}

template <typename X, typename W, int VEC, int ITER, int LANES, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) layer_norm_bwd_kernel(const __grid_constant__ Params p) {
    chain_wait();
    constexpr int GROUPS = THREADS / LANES;
    using R = Ring<X, VEC, ITER, LANES, THREADS, 2>;
    using L = Lane<VEC>;
    typedef typename L::T T;
    __shared__ float sh[2][2][THREADS / 32];
    extern __shared__ __align__(16) unsigned char ring_raw[];
    X* ring = reinterpret_cast<X*>(ring_raw);
    float* cols = reinterpret_cast<float*>(ring_raw);     // [2][N], after the last row
    const int N = p.N, lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.f / (float)N;
    const X *x = static_cast<const X*>(p.x), *dy = static_cast<const X*>(p.dy);
    X* dx = static_cast<X*>(p.dx);
    const W* w = static_cast<const W*>(p.w);
    const long stride = (long)gridDim.x * GROUPS, first = (long)blockIdx.x * GROUPS + group;
    const auto fetch = [&](long row, int stage) {
        if (row < p.rows) {
            R::bring(ring, stage, 0, x, row, p.rows, N, lane);
            R::bring(ring, stage, 1, dy, row, p.rows, N, lane);
        }
        copies_commit();
    };
#pragma unroll
    for (int k = 0; k < R::STAGES - 1; ++k) fetch(first + k * stride, k);
    T dw[ITER][L::N], db[ITER][L::N], wv[ITER][L::N];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * LANES + lane) * VEC;
#pragma unroll
        for (int u = 0; u < L::N; ++u) {
            dw[i][u] = db[i][u] = splat<T>(0.f);
            wv[i][u] = splat<T>(1.f);
        }
        if (w && c < N) L::load(w + c, wv[i]);
    }
    float mean = first < p.rows ? p.mean[first] : 0.f, rstd = first < p.rows ? p.rstd[first] : 0.f;
    int stage = 0, par = 0;
    for (long row = first; row - group < p.rows; row += stride, par ^= 1, stage = stage + 1 == R::STAGES ? 0 : stage + 1) {
        copies_but<R::STAGES - 2>();
        if constexpr (R::SHARED) __syncthreads();
        T xh[ITER][L::N], d[ITER][L::N];
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (row < p.rows && (i * LANES + lane) * VEC < N) {
                R::read(ring, stage, i, 0, row, N, lane, xh[i]);
                R::read(ring, stage, i, 1, row, N, lane, d[i]);
            } else {
#pragma unroll
                for (int u = 0; u < L::N; ++u) xh[i][u] = d[i][u] = splat<T>(0.f);      // (d of zero adds nothing)
            }
        }
        fetch(row + (R::STAGES - 1) * stride, stage == 0 ? R::STAGES - 1 : stage - 1);
        const T neg = splat<T>(-mean), r = splat<T>(rstd);
        if (row + stride < p.rows) {
            mean = p.mean[row + stride];
            rstd = p.rstd[row + stride];
        }
        T s0 = splat<T>(0.f), s1 = s0;
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int u = 0; u < L::N; ++u) {
                xh[i][u] = mul(add(xh[i][u], neg), r);
                dw[i][u] = fma2(d[i][u], xh[i][u], dw[i][u]);
                db[i][u] = add(db[i][u], d[i][u]);
                d[i][u] = mul(d[i][u], wv[i][u]);
                s0 = add(s0, d[i][u]);
                s1 = fma2(d[i][u], xh[i][u], s1);
            }
        float s[2] = {total(s0), total(s1)};
        row_sum<LANES, THREADS>(s, sh[par]);
        // rstd (z - mean(z) - xhat mean(z xhat))
        const T m1 = splat<T>(-s[0] * inv), m2 = splat<T>(-s[1] * inv);
        if (row < p.rows) {
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                const int c = (i * LANES + lane) * VEC;
                if (c < N) {
#pragma unroll
                    for (int u = 0; u < L::N; ++u) d[i][u] = mul(fma2(xh[i][u], m2, add(d[i][u], m1)), r);
                    L::store(dx + row * N + c, d[i]);
                }
            }
        }
    }
    if (!p.part) return;
    copies_but<0>();
    __syncthreads();
    float* part = p.part + (long)blockIdx.x * 2 * N;
    if constexpr (GROUPS == 1) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * LANES + lane) * VEC;
            if (c < N) {
                L::store(part + c, dw[i]);
                L::store(part + N + c, db[i]);
            }
        }
    } else {
        // the groups in turn
        for (int g = 0; g < GROUPS; ++g) {
            __syncthreads();
            if (group == g) {
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
                    const int c = (i * LANES + lane) * VEC;
                    if (c < N) {
                        if (g) {
                            T a[L::N], e[L::N];
                            L::load(cols + c, a);
                            L::load(cols + N + c, e);
#pragma unroll
                            for (int u = 0; u < L::N; ++u) {
                                dw[i][u] = add(a[u], dw[i][u]);
                                db[i][u] = add(e[u], db[i][u]);
                            }
                        }
                        L::store(cols + c, dw[i]);
                        L::store(cols + N + c, db[i]);
                    }
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * N; i += THREADS) part[i] = cols[i];
    }
}

// ---- rows of any length: 256 threads a row, read again for each sum
template <int V>
__device__ __forceinline__ void wide_sum(float (&s)[V], float (*sh)[8]) {
    row_sum<256, 256>(s, sh);
    __syncthreads();
}
template <typename X, typename W>
__global__ void __launch_bounds__(256) layer_norm_wide_fwd_kernel(const __grid_constant__ Params p) {
    chain_wait();
    __shared__ float sh[1][8];
    const int N = p.N;
    const float inv = 1.f / (float)N;
    const long row = blockIdx.x;
    const X* x = static_cast<const X*>(p.x) + row * N;
    X* y = static_cast<X*>(p.y) + row * N;
    const W *w = static_cast<const W*>(p.w), *b = static_cast<const W*>(p.b);
    float s[1] = {0.f}, ss[1] = {0.f};
    for (int i = threadIdx.x; i < N; i += 256) s[0] += get(x + i);
    wide_sum(s, sh);
    const float mean = s[0] * inv;
    for (int i = threadIdx.x; i < N; i += 256) {
        const float d = get(x + i) - mean;
        ss[0] = fmaf(d, d, ss[0]);
    }
    wide_sum(ss, sh);
    const float rstd = rsqrtf(ss[0] * inv + p.eps);
    for (int i = threadIdx.x; i < N; i += 256) {
        float v = (get(x + i) - mean) * rstd;
        if (w) v *= get(w + i);
        if (b) v += get(b + i);
        put(y + i, v);
    }
    if (threadIdx.x == 0 && p.mean) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
}
template <typename X, typename W>
__global__ void __launch_bounds__(256) layer_norm_wide_dx_kernel(const __grid_constant__ Params p) {
    chain_wait();
    __shared__ float sh[2][8];
    const int N = p.N;
    const float inv = 1.f / (float)N;
    const long row = blockIdx.x;
    const X *x = static_cast<const X*>(p.x) + row * N, *dy = static_cast<const X*>(p.dy) + row * N;
    X* dx = static_cast<X*>(p.dx) + row * N;
    const W* w = static_cast<const W*>(p.w);
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int i = threadIdx.x; i < N; i += 256) {
        const float z = w ? get(dy + i) * get(w + i) : get(dy + i);
        s[0] += z;
        s[1] = fmaf(z, (get(x + i) - mean) * rstd, s[1]);
    }
    wide_sum(s, sh);
    for (int i = threadIdx.x; i < N; i += 256) {
        const float z = w ? get(dy + i) * get(w + i) : get(dy + i), xhat = (get(x + i) - mean) * rstd;
        put(dx + i, rstd * (z - s[0] * inv - xhat * (s[1] * inv)));
    }
}
// partial sums over every parts-th row, a thread a column
template <typename X>
__global__ void __launch_bounds__(256) layer_norm_wide_columns_kernel(const __grid_constant__ Params p) {
    chain_wait();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.N) return;
    const X *x = static_cast<const X*>(p.x), *dy = static_cast<const X*>(p.dy);
    float dw = 0.f, db = 0.f;
    for (long row = blockIdx.y; row < p.rows; row += p.parts) {
        const float d = get(dy + row * p.N + c);
        dw = fmaf(d, (get(x + row * p.N + c) - p.mean[row]) * p.rstd[row], dw);
        db += d;
    }
    p.part[(long)blockIdx.y * 2 * p.N + c] = dw;
    p.part[((long)blockIdx.y * 2 + 1) * p.N + c] = db;
}

// dw and db of 32 columns a CTA: 32 warps take the parts in turn, four in flight each, then the warps' sums
template <typename W>
__global__ void __launch_bounds__(1024) layer_norm_gather_kernel(const __grid_constant__ Params p) {
    chain_wait();
    __shared__ float sh[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long c = (long)blockIdx.x * 32 + lane;          // of the 2 N of a part
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < 2l * p.N)
        for (int i = warp; i < p.parts; i += 128)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + 32 * u < p.parts) s[u] += p.part[(long)(i + 32 * u) * 2 * p.N + c];
    sh[warp][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    // a warp a column, a lane a warp's sum
    float t = sh[lane][warp];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    const long at = (long)blockIdx.x * 32 + warp;
    if (lane == 0 && at < 2l * p.N) {
        if (at < p.N) {
            if (p.dw) put(static_cast<W*>(p.dw) + at, t);
        } else if (p.db) {
            put(static_cast<W*>(p.db) + at - p.N, t);
        }
    }
}

// ---- which kernel: a row in the registers of LANES lanes, ITER words of VEC values each
template <typename KernT>
cudaError_t run(KernT kern, dim3 grid, int threads, size_t smem, const Params& p, cudaStream_t st) {
    if (smem > 0) {
        const cudaError_t e = allow_smem(kern, smem);
        if (e != cudaSuccess) return e;
    }
    const cudaError_t e = launch_chained(kern, grid, threads, smem, st, p);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return e;
}
// Lanes a row, so that each has `values` of it; a power of two of at least a warp and at most the CTA.
constexpr int SMS = 148, MAX_N = 8192;
int lanes_of(int N, int values, int threads) {
    int lanes = 32;
    while (lanes * values < N && lanes < threads) lanes *= 2;
    return lanes;
}
int ctas_of(long rows, int groups, int per_sm) {
    const long n = (rows + groups - 1) / groups;
    return (int)(n < per_sm * SMS ? n : per_sm * SMS);
}
// Forward: 16 values a lane, two CTAs of 256 threads an SM (32768 x 2048 bf16, us: 51; 8 values in two CTAs of 512 59, 16 in one of 512 59, 16 in three of 256 51, 32 in two
// of 256 49, but there 16384 x 4096 fp32 and short rows lose).  Backward: 32 bytes of a row a lane, one CTA of 512 (82; 16 bytes of one row 111, of two rows at once
// 92..100, 32 bytes in two CTAs of 256 80, in three 133).  The longest rows have twice that a lane.
constexpr int FWD_THREADS = 256, FWD_VALUES = 16, BWD_THREADS = 512;
constexpr int bwd_values(size_t bytes) { return 32 / (int)bytes; }
int parts_of(long rows, int N, int bytes) {
    if (N > MAX_N) return (int)(rows < 64 ? rows : 64);
    return ctas_of(rows, BWD_THREADS / lanes_of(N, bwd_values(bytes), BWD_THREADS), 1);
}
template <typename X, typename W, int VEC, int ITER, int LANES>
cudaError_t fwd_pass(const Params& p, cudaStream_t st) {
    return run(layer_norm_fwd_kernel<X, W, VEC, ITER, LANES, FWD_THREADS>, ctas_of(p.rows, FWD_THREADS / LANES, 2), FWD_THREADS,
               Ring<X, VEC, ITER, LANES, FWD_THREADS, 1>::SIZE, p, st);
}
template <typename X, typename W, int VEC, int ITER, int LANES>
cudaError_t bwd_pass(const Params& p, cudaStream_t st) {
    return run(layer_norm_bwd_kernel<X, W, VEC, ITER, LANES, BWD_THREADS>, p.parts, BWD_THREADS, Ring<X, VEC, ITER, LANES, BWD_THREADS, 2>::SIZE, p, st);
}
template <typename X, typename W, int VEC>
cudaError_t fwd_vec(const Params& p, cudaStream_t st) {
    constexpr int I = FWD_VALUES / VEC, MOST = MAX_N / FWD_THREADS / VEC;
    switch (lanes_of(p.N, FWD_VALUES, FWD_THREADS)) {
        case 32:                                            // short rows: no more than they have
            if (VEC <= 4 && p.N <= 4 * 32) return fwd_pass<X, W, VEC, (VEC <= 4 ? 4 / VEC : 1), 32>(p, st);
            return p.N <= 8 * 32 ? fwd_pass<X, W, VEC, 8 / VEC, 32>(p, st) : fwd_pass<X, W, VEC, I, 32>(p, st);
        case 64: return fwd_pass<X, W, VEC, I, 64>(p, st);
        case 128: return fwd_pass<X, W, VEC, I, 128>(p, st);
        default: return p.N <= FWD_VALUES * FWD_THREADS ? fwd_pass<X, W, VEC, I, FWD_THREADS>(p, st) : fwd_pass<X, W, VEC, MOST, FWD_THREADS>(p, st);
    }
}
template <typename X, typename W, int VEC>
cudaError_t bwd_vec(const Params& p, cudaStream_t st) {
    constexpr int V = bwd_values(sizeof(X)), I = V / VEC, MOST = MAX_N / BWD_THREADS / VEC;
    switch (lanes_of(p.N, V, BWD_THREADS)) {
        case 32:
            if (VEC <= 4 && p.N <= 4 * 32) return bwd_pass<X, W, VEC, (VEC <= 4 ? 4 / VEC : 1), 32>(p, st);
            return p.N <= 8 * 32 ? bwd_pass<X, W, VEC, 8 / VEC, 32>(p, st) : bwd_pass<X, W, VEC, I, 32>(p, st);
        case 64: return bwd_pass<X, W, VEC, I, 64>(p, st);
        case 128: return bwd_pass<X, W, VEC, I, 128>(p, st);
        case 256: return bwd_pass<X, W, VEC, I, 256>(p, st);
        default: return p.N <= V * BWD_THREADS ? bwd_pass<X, W, VEC, I, BWD_THREADS>(p, st) : bwd_pass<X, W, VEC, MOST, BWD_THREADS>(p, st);
    }
}
template <typename X, typename W>
cudaError_t rows_in_registers(bool back, const Params& p, cudaStream_t st) {
    constexpr int VEC = 16 / (int)sizeof(X);
    if (back) return p.N % VEC == 0 ? bwd_vec<X, W, VEC>(p, st) : bwd_vec<X, W, 1>(p, st);
    return p.N % VEC == 0 ? fwd_vec<X, W, VEC>(p, st) : fwd_vec<X, W, 1>(p, st);
}
template <typename X, typename W>
cudaError_t forward(const Params& p, cudaStream_t st) {
    if (p.N > MAX_N) return run(layer_norm_wide_fwd_kernel<X, W>, (unsigned)p.rows, 256, 0, p, st);
    return rows_in_registers<X, W>(false, p, st);
}
template <typename X, typename W>
cudaError_t backward(Params p, cudaStream_t st) {
    const bool sums = p.dw || p.db;
    if (!sums) p.part = nullptr;
    cudaError_t e;
    if (p.N > MAX_N) {
        e = run(layer_norm_wide_dx_kernel<X, W>, (unsigned)p.rows, 256, 0, p, st);
        if (e == cudaSuccess && sums) e = run(layer_norm_wide_columns_kernel<X>, dim3((p.N + 255) / 256, p.parts), 256, 0, p, st);
    } else {
        e = rows_in_registers<X, W>(true, p, st);
    }
    if (e == cudaSuccess && sums) e = run(layer_norm_gather_kernel<W>, (unsigned)((2l * p.N + 31) / 32), 1024, 0, p, st);
    return e;
}
int check(int x_f32, int w_f32, long rows, int N) {
    // (columns are counted in ints, a stride behind the row's end)
    if (rows < 1 || N < 1 || rows > 0x7fffffffl || N > 1 << 30 || (x_f32 && !w_f32)) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    return 0;
}

}  // namespace norm
}  // namespace llattn

using namespace llattn;

extern "C" {

size_t llattn_layer_norm_bwd_workspace_bytes(long rows, int N) {
    if (norm::check(0, 0, rows, N) != 0) return 0;
    return (size_t)norm::parts_of(rows, N, 4) * 2 * N * sizeof(float);       // (of either type: fp32 rows have the more parts)
}

int llattn_layer_norm_fwd(const void* x, int x_is_f32, const void* w, const void* b, int w_is_f32, void* y, float* mean, float* rstd, float eps, long rows,
                          int N, void* stream) {
    const int rc = norm::check(x_is_f32, w_is_f32, rows, N);
    if (rc != 0) return rc;
    if (!x || !y || (mean && !rstd) || (rstd && !mean)) return LLATTN_ERR_NULL;
    if (misaligned(16, {x, w, b, y, mean, rstd})) return LLATTN_ERR_ALIGNMENT;
    norm::Params p = {};
    p.x = x;
    p.w = w;
    p.b = b;
    p.y = y;
    p.mean = mean;
    p.rstd = rstd;
    p.rows = rows;
    p.N = N;
    p.eps = eps;
    cudaStream_t st = (cudaStream_t)stream;
    if (x_is_f32) return (int)norm::forward<float, float>(p, st);
    return (int)(w_is_f32 ? norm::forward<norm::bf16, float>(p, st) : norm::forward<norm::bf16, norm::bf16>(p, st));
}

int llattn_layer_norm_bwd(const void* x, int x_is_f32, const void* w, int w_is_f32, const float* mean, const float* rstd, const void* dy, void* dx, void* dw,
                          void* db, void* workspace, size_t workspace_bytes, long rows, int N, void* stream) {
    const int rc = norm::check(x_is_f32, w_is_f32, rows, N);
    if (rc != 0) return rc;
    if (!x || !mean || !rstd || !dy || !dx) return LLATTN_ERR_NULL;
    if (misaligned(16, {x, w, mean, rstd, dy, dx, dw, db})) return LLATTN_ERR_ALIGNMENT;
    if ((dw || db) && (!workspace || misaligned(256, {workspace}) || workspace_bytes < llattn_layer_norm_bwd_workspace_bytes(rows, N))) return LLATTN_ERR_WORKSPACE;
    norm::Params p = {};
    p.x = x;
    p.w = w;
    p.dy = dy;
    p.dx = dx;
    p.dw = dw;
    p.db = db;
    p.mean = const_cast<float*>(mean);
    p.rstd = const_cast<float*>(rstd);
    p.part = static_cast<float*>(workspace);
    p.rows = rows;
    p.N = N;
    p.parts = norm::parts_of(rows, N, x_is_f32 ? 4 : 2);
    cudaStream_t st = (cudaStream_t)stream;
    if (x_is_f32) return (int)norm::backward<float, float>(p, st);
    return (int)(w_is_f32 ? norm::backward<norm::bf16, float>(p, st) : norm::backward<norm::bf16, norm::bf16>(p, st));
}

}  // extern "C"
