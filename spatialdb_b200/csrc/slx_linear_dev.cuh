// slx_linear_dev.cuh -- element types and the epilogue shared by the linear operator's kernels.
#pragma once
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace slx {
namespace lin {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU_TANH = 3, ACT_GELU_ERF = 4 };

// The activations in fp32, for the output type T. For f32 outputs they call the full-precision expf and erff;
// a 16-bit output's half step (2^-9 or 2^-12 of it) leaves room for the hardware exponential (a few units of
// 2^-22) and for Abramowitz and Stegun's 7.1.26, erf(z) = 1 - (a1 t + ... + a5 t^5) e^(-z^2) with
// t = 1 / (1 + 0.3275911 z), whose error is at most 1.5e-7. Quotients round to 2 units; one whose divisor
// passes 2^126 becomes 0, an absolute error below 2^-118. ReLU keeps a NaN.
template <class T>
__device__ __forceinline__ float exp_for(float v) {
    return sizeof(T) == 4 ? expf(v) : __expf(v);
}
template <class T>
__device__ __forceinline__ float silu_for(float v, float s) {  // v / (1 + e^-s)
    return __fdividef(v, 1.0f + exp_for<T>(-s));
}
template <class T, int ACT>
__device__ __forceinline__ float activate(float v) {
    if (ACT == ACT_RELU) return v < 0.0f ? 0.0f : v;
    if (ACT == ACT_SILU) return silu_for<T>(v, v);
    if (ACT == ACT_GELU_TANH)  // 0.5 (1 + tanh u) = 1 / (1 + e^-2u)
        return silu_for<T>(v, 1.5957691216057308f * fmaf(0.044715f * v * v, v, v));
    if (ACT == ACT_GELU_ERF) {
        if (sizeof(T) == 4) return 0.5f * v * (1.0f + erff(v * 0.7071067811865476f));
        const float z = fabsf(v) * 0.7071067811865476f;
        const float t = __fdividef(1.0f, fmaf(0.3275911f, z, 1.0f));
        const float s = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
        const float tail = 0.5f * s * __expf(-z * z);  // (1 - erf z) / 2
        return v * (v < 0.0f ? tail : 1.0f - tail);
    }
    return v;
}
template <class T, int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act) {
    switch (act) {
        case ACT_RELU:
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = activate<T, ACT_RELU>(v[j]);
            break;
        case ACT_SILU:
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = activate<T, ACT_SILU>(v[j]);
            break;
        case ACT_GELU_TANH:
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = activate<T, ACT_GELU_TANH>(v[j]);
            break;
        case ACT_GELU_ERF:
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = activate<T, ACT_GELU_ERF>(v[j]);
            break;
        default: break;
    }
}

}  // namespace lin
}  // namespace slx
