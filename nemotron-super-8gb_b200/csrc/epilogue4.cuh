// The epilogue of the four-bit linear, shared by its kernels.
#pragma once
#include "common.cuh"

namespace qmoe {
namespace g4 {

// Results. The linear's value is rounded to the output type, then (in fp32, rounded again) its squared ReLU or the sum
// with the residual, as the unfused operators round (no fused multiply-add). EPI is a template argument and its switch
// stands outside the unrolled columns: with it inside, the epilogue's code no longer fitted the instruction cache and
// 32 columns took 2,400 cycles instead of 200.
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float wide(__half v) { return __half2float(v); }

// sx * sw * v and its epilogue, before the last rounding.
template <typename T, int EPI> __device__ __forceinline__ float finish(float v, float sx, float sw, float res) {
    v = __fmul_rn(__fmul_rn(v, sx), sw);
    if (EPI == 1) {
        float r;
        asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(wide(narrow<T>(v))));   // relu, NaN kept
        return __fmul_rn(r, r);
    }
    return EPI == 2 ? __fadd_rn(wide(narrow<T>(v)), res) : v;
}

template <typename T, int EPI> __device__ __forceinline__ void store_one(void *y, const void *res, int64_t at, float v, float sx, float sw) {
    static_cast<T *>(y)[at] = narrow<T>(finish<T, EPI>(v, sx, sw, EPI == 2 ? wide(static_cast<const T *>(res)[at]) : 0.f));
}

} // namespace g4
} // namespace qmoe
