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

// The activations in fp32, for the output type T: v times a factor that is small in the negative tail and is formed
// without cancellation, so that the result is good to a few roundings of itself there too. f32 outputs call expf; a
// 16-bit output's half step (2^-12 or 2^-9 of it) leaves room for the hardware's exponential (2 + 1.2 |s| units of
// 2^-23) and reciprocal, and for a shorter polynomial in the complementary error function. ReLU keeps a NaN.
template <class T>
__device__ __forceinline__ float exp_for(float v) {
    return sizeof(T) == 4 ? expf(v) : __expf(v);
}
// a / b for 0 <= a <= 1 <= b: f32 to one rounding (a corrected reciprocal, b below 2^126), 16-bit outputs to two units.
template <class T>
__device__ __forceinline__ float over(float a, float b) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(b));
    const float q = a * r;
    return sizeof(T) == 4 ? fmaf(fmaf(-b, q, a), r, q) : q;
}
template <class T>
__device__ __forceinline__ float logistic_times(float v, float s) {  // v / (1 + e^-s) from e^-|s|, which does not overflow
    const float t = exp_for<T>(-fabsf(s));
    return v * over<T>(s < 0.0f ? t : 1.0f, 1.0f + t);
}
// erfc(|v| / sqrt(2)) / 2 = e^(-v^2 / 2) t P(t), t = 1 / (1 + a z), z = |v| / sqrt(2): P has the least relative error of
// its degree (iterated weighted least squares over Chebyshev points, then steps of fp32 coefficients) wherever the
// outputs' type can hold the result, 2.7e-8 for z <= 10.2 in f32, 5.2e-6 (2^-17.5) for z <= 9.6 in 16 bits. With
// CUDA's erfcf bf16 8192 x 768 x 2304 takes 59 us in place of 36.
template <class T>
__device__ __forceinline__ float erfc_half(float v) {
    constexpr bool F = sizeof(T) == 4;
    constexpr float A = F ? 0.3f : 0.44f;
    constexpr float c32[9] = {0.169187695f, 0.170719847f, 0.148310736f, 0.215023339f, -0.0948533937f, 0.547983646f, -0.512487233f, 0.485655934f, -0.129540592f};
    constexpr float c16[6] = {0.248561069f, 0.242569029f, 0.26358822f, 0.0407278016f, 0.350655288f, -0.146106571f};
    const float z = 0.7071067811865476f * (F ? fminf(fabsf(v), 64.0f) : fabsf(v));  // past 64 the exponential is zero
    const float t = over<T>(1.0f, fmaf(A, z, 1.0f));
    float c = F ? c32[8] : c16[5];
#pragma unroll
    for (int i = F ? 7 : 4; i >= 0; i--) c = fmaf(t, c, F ? c32[i] : c16[i < 6 ? i : 5]);
    return 0.5f * t * c * exp_for<T>(-0.5f * v * v);
}
template <class T, int ACT>
__device__ __forceinline__ float activate(float v) {
    if (ACT == ACT_RELU) return v < 0.0f ? 0.0f : v;
    if (ACT == ACT_SILU) return logistic_times<T>(v, v);
    if (ACT == ACT_GELU_TANH)  // 0.5 (1 + tanh u) = 1 / (1 + e^-2u)
        return logistic_times<T>(v, 1.5957691216057308f * fmaf(0.044715f * v * v, v, v));
    if (ACT == ACT_GELU_ERF) {  // v (1 + erf(v / sqrt(2))) / 2
        const float tail = erfc_half<T>(v);
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
