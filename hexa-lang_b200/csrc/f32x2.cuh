// f32x2.cuh — pairs of fp32 in a 64-bit register with sm_100's two-lane
// instructions (one issue slot for two results), and the hardware exp2 and
// three-input maximum.
#pragma once
#include <cuda_runtime.h>

// 2^x, relative error about 2^-22; denormal results are 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
struct F2 {
    float2 v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float2 w) { v = w; }
    __device__ __forceinline__ F2(float x, float y) { v = make_float2(x, y); }
    __device__ __forceinline__ float x() const { return v.x; }
    __device__ __forceinline__ float y() const { return v.y; }
};
__device__ __forceinline__ F2 operator+(F2 a, F2 b) { return __fadd2_rn(a.v, b.v); }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) { return __fmul2_rn(a.v, b.v); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { return __ffma2_rn(a.v, b.v, c.v); }
