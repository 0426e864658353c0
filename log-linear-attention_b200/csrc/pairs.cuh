// Two fp32 values in one 64-bit register (the f32x2 instructions), and the same operations on single values, for kernels that are written for either.
#pragma once
#include <stdint.h>

namespace llattn {

struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 pair(float lo, float hi) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 both(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 add(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float fma2(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float total(F2 a) {
    const float2 f = both(a);
    return f.x + f.y;
}
__device__ __forceinline__ float total(float a) { return a; }
template <typename T>
__device__ __forceinline__ T splat(float a);
template <>
__device__ __forceinline__ float splat<float>(float a) { return a; }
template <>
__device__ __forceinline__ F2 splat<F2>(float a) { return pair(a, a); }
__device__ __forceinline__ F2 shfl_up(F2 a, int d) { return F2{__shfl_up_sync(0xffffffffu, a.v, d)}; }
__device__ __forceinline__ F2 shfl_down(F2 a, int d) { return F2{__shfl_down_sync(0xffffffffu, a.v, d)}; }
__device__ __forceinline__ float shfl_up(float a, int d) { return __shfl_up_sync(0xffffffffu, a, d); }
__device__ __forceinline__ float shfl_down(float a, int d) { return __shfl_down_sync(0xffffffffu, a, d); }

}  // namespace llattn
