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

// 2^x and 1 / x by the hardware (relative errors near 2^-22); infinities give 0.
__device__ __forceinline__ float ex2_f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_f(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.4426950408889634f;

// act(z) = z s, and s for the slope; t = z^2 is held at 400 (|z| = 20, where s is
// 0 or 1 to the last bit), so that no product of infinities with zeros can arise.
__device__ __forceinline__ float act_sigmoid(float z, int act, float& t) {
    if (act == Q6_ACT_GELU_TANH) {
        t = fminf(z * z, 400.0f);
        return rcp_f(1.0f + ex2_f(z * fmaf(t, -kLog2e * kGelu2K * kGeluC, -kLog2e * kGelu2K)));
    }
    return rcp_f(1.0f + ex2_f(-kLog2e * z));
}

__device__ __forceinline__ float act_f(float z, int act) {
    if (act == Q6_ACT_NONE) return z;
    float t;
    return z * act_sigmoid(z, act, t);
}

// act(z) and act'(z) = s + z s (1 - s) du/dz, u the sigmoid's argument.
__device__ __forceinline__ void act_and_slope_f(float z, int act, float& a, float& slope) {
    if (act == Q6_ACT_NONE) {
        a = z;
        slope = 1.0f;
        return;
    }
    float t;
    const float s = act_sigmoid(z, act, t);
    a = z * s;
    const float q = a * (1.0f - s);
    slope = act == Q6_ACT_GELU_TANH ? fmaf(q, fmaf(t, 3.0f * kGelu2K * kGeluC, kGelu2K), s) : q + s;
}

// 16-byte (or smaller) read-only loads: free to move across stores.
template <typename S>
__device__ __forceinline__ S load_ro(const void* p) {
    static_assert(sizeof(S) == 2 || sizeof(S) == 4 || sizeof(S) == 8 || sizeof(S) % 16 == 0, "load size");
    S out;
    if constexpr (sizeof(S) % 16 == 0) {
        uint4* o = reinterpret_cast<uint4*>(&out);
#pragma unroll
        for (int i = 0; i < int(sizeof(S) / 16); ++i) o[i] = __ldg(static_cast<const uint4*>(p) + i);
    } else if constexpr (sizeof(S) == 8) {
        *reinterpret_cast<uint2*>(&out) = __ldg(static_cast<const uint2*>(p));
    } else if constexpr (sizeof(S) == 4) {
        *reinterpret_cast<uint32_t*>(&out) = __ldg(static_cast<const uint32_t*>(p));
    } else {
        *reinterpret_cast<uint16_t*>(&out) = __ldg(static_cast<const uint16_t*>(p));
    }
    return out;
}

}  // namespace q6
