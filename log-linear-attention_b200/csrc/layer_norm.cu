// Layer norm over rows of N values and its gradients:
//     y  = (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//     dx = rstd (z - mean(z) - xhat mean(z xhat)),   z = w dy,  xhat = (x - mean) rstd
//     dw = sum over rows of dy xhat,   db = sum over rows of dy
// w absent is ones, b absent zeros.  All sums in fp32; the variance from the differences to the mean.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/llattn.h"
#include "launch_count.h"

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

// sums of a and b over the CTA's 256 threads
__device__ __forceinline__ float2 cta_sum(float a, float b, float2* sh) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, d);
        b += __shfl_xor_sync(0xffffffffu, b, d);
    }
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        s.x += sh[w].x;
        s.y += sh[w].y;
    }
    __syncthreads();
    return s;
}

template <typename X, typename W>
__global__ void __launch_bounds__(256) layer_norm_fwd_kernel(const __grid_constant__ Params p) {
    chain_wait();
    __shared__ float2 sh[8];
    const int N = p.N;
    const float inv = 1.f / (float)N;
    const long row = blockIdx.x;
    const X* x = static_cast<const X*>(p.x) + row * N;
    X* y = static_cast<X*>(p.y) + row * N;
    const W *w = static_cast<const W*>(p.w), *b = static_cast<const W*>(p.b);
    float s = 0.f, ss = 0.f;
    for (int i = threadIdx.x; i < N; i += 256) s += get(x + i);
    const float mean = cta_sum(s, 0.f, sh).x * inv;
    for (int i = threadIdx.x; i < N; i += 256) {
        const float d = get(x + i) - mean;
        ss = fmaf(d, d, ss);
    }
    const float rstd = rsqrtf(cta_sum(ss, 0.f, sh).x * inv + p.eps);
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
__global__ void __launch_bounds__(256) layer_norm_dx_kernel(const __grid_constant__ Params p) {
    chain_wait();
    __shared__ float2 sh[8];
    const int N = p.N;
    const float inv = 1.f / (float)N;
    const long row = blockIdx.x;
    const X *x = static_cast<const X*>(p.x) + row * N, *dy = static_cast<const X*>(p.dy) + row * N;
    X* dx = static_cast<X*>(p.dx) + row * N;
    const W* w = static_cast<const W*>(p.w);
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s = 0.f, sx = 0.f;
    for (int i = threadIdx.x; i < N; i += 256) {
        const float z = w ? get(dy + i) * get(w + i) : get(dy + i);
        s += z;
        sx = fmaf(z, (get(x + i) - mean) * rstd, sx);
    }
    const float2 m = cta_sum(s, sx, sh);
    for (int i = threadIdx.x; i < N; i += 256) {
        const float z = w ? get(dy + i) * get(w + i) : get(dy + i), xhat = (get(x + i) - mean) * rstd;
        put(dx + i, rstd * (z - m.x * inv - xhat * (m.y * inv)));
    }
}

// partial sums over every parts-th row, a thread a column
template <typename X>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const __grid_constant__ Params p) {
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

template <typename W>
__global__ void __launch_bounds__(256) layer_norm_gather_kernel(const __grid_constant__ Params p) {
    chain_wait();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.N) return;
    float dw = 0.f, db = 0.f;
    for (int i = 0; i < p.parts; ++i) {
        dw += p.part[(long)i * 2 * p.N + c];
        db += p.part[((long)i * 2 + 1) * p.N + c];
    }
    if (p.dw) put(static_cast<W*>(p.dw) + c, dw);
    if (p.db) put(static_cast<W*>(p.db) + c, db);
}

int parts_of(long rows) { return (int)(rows < 64 ? rows : 64); }

template <typename X, typename W>
cudaError_t forward(const Params& p, cudaStream_t st) {
    const cudaError_t e = launch_chained(layer_norm_fwd_kernel<X, W>, (unsigned)p.rows, 256, 0, st, p);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return e;
}
template <typename X, typename W>
cudaError_t backward(const Params& p, cudaStream_t st) {
    cudaError_t e = launch_chained(layer_norm_dx_kernel<X, W>, (unsigned)p.rows, 256, 0, st, p);
    if (e != cudaSuccess) return e;
    LLATTN_LAUNCHED();
    if (!p.dw && !p.db) return e;
    const unsigned blocks = (p.N + 255) / 256;
    e = launch_chained(layer_norm_columns_kernel<X>, dim3(blocks, p.parts), 256, 0, st, p);
    if (e != cudaSuccess) return e;
    LLATTN_LAUNCHED();
    e = launch_chained(layer_norm_gather_kernel<W>, blocks, 256, 0, st, p);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return e;
}
int check(int x_f32, int w_f32, long rows, int N) {
    if (rows < 1 || N < 1 || rows > 0x7fffffffl || (x_f32 && !w_f32)) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    return 0;
}

}  // namespace norm
}  // namespace llattn

using namespace llattn;

extern "C" {

size_t llattn_layer_norm_bwd_workspace_bytes(long rows, int N) {
    if (norm::check(0, 0, rows, N) != 0) return 0;
    return (size_t)norm::parts_of(rows) * 2 * N * sizeof(float);
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
    p.parts = norm::parts_of(rows);
    cudaStream_t st = (cudaStream_t)stream;
    if (x_is_f32) return (int)norm::backward<float, float>(p, st);
    return (int)(w_is_f32 ? norm::backward<norm::bf16, float>(p, st) : norm::backward<norm::bf16, norm::bf16>(p, st));
}

}  // extern "C"
