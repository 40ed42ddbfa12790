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

// The activation in fp32. The comparison in ReLU keeps a NaN.
__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case ACT_RELU: return v < 0.0f ? 0.0f : v;
        case ACT_SILU: return v / (1.0f + expf(-v));
        case ACT_GELU_TANH: {
            const float u = 0.7978845608028654f * fmaf(0.044715f * v * v, v, v);
            return 0.5f * v * (1.0f + tanhf(u));
        }
        case ACT_GELU_ERF: return 0.5f * v * (1.0f + erff(v * 0.7071067811865476f));
        default: return v;
    }
}

}  // namespace lin
}  // namespace slx
