// Device helpers of the dense linear and the layer norm: element types,
// 16-byte groups of eight elements, activations and their derivatives.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "q6_b200.h"

namespace q6 {

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }

// The activations as z sigmoid(s): GELU-tanh is z sigmoid(2 u) because
// (1 + tanh u) / 2 = sigmoid(2 u).  In this form small outputs of negative z
// keep their relative accuracy (1 + tanh cancels there).  exp overflowing to
// infinity gives sigmoid 0.
constexpr float kGelu2K = 2.0f * 0.7978845608028654f;  // 2 sqrt(2 / pi)
constexpr float kGeluC = 0.044715f;

__device__ __forceinline__ float sigmoid_f(float s) { return __fdividef(1.0f, 1.0f + __expf(-s)); }

__device__ __forceinline__ float act_f(float z, int act) {
    if (act == Q6_ACT_GELU_TANH) return z * sigmoid_f(kGelu2K * z * fmaf(kGeluC * z, z, 1.0f));
    if (act == Q6_ACT_SILU) return z * sigmoid_f(z);
    return z;
}

// act(z) and act'(z) = s + z s (1 - s) ds/dz.  Beyond |z| = 12 the second term
// is below 1e-30 for GELU; z is held there so that z^2 cannot overflow into 0 * inf.
__device__ __forceinline__ void act_and_slope_f(float z, int act, float& a, float& slope) {
    if (act == Q6_ACT_GELU_TANH) {
        const float s = sigmoid_f(kGelu2K * z * fmaf(kGeluC * z, z, 1.0f));
        const float h = fminf(fmaxf(z, -12.0f), 12.0f);
        a = z * s;
        slope = fmaf(h * s * (1.0f - s), kGelu2K * fmaf(3.0f * kGeluC * h, h, 1.0f), s);
    } else if (act == Q6_ACT_SILU) {
        const float s = sigmoid_f(z);
        a = z * s;
        slope = fmaf(z * (1.0f - s), s, s);
    } else {
        a = z;
        slope = 1.0f;
    }
}

}  // namespace q6
