// Device helpers of the dense linear and the layer norm: element types,
// 16-byte groups of eight elements, activations and their derivatives.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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
        t = fminf(__fmul_rn(z, z), 400.0f);
        return rcp_f(__fadd_rn(1.0f, ex2_f(__fmul_rn(z, fmaf(t, -kLog2e * kGelu2K * kGeluC, -kLog2e * kGelu2K)))));
    }
    return rcp_f(__fadd_rn(1.0f, ex2_f(__fmul_rn(-kLog2e, z))));
}

// The epilogue's steps are written with explicit roundings (here and below): left
// to the compiler, a product and a sum may or may not become one operation, by
// what else a kernel writes, and a forward pass with and without gradients would
// differ in its last bits.
__device__ __forceinline__ float act_f(float z, int act) {
    if (act == Q6_ACT_NONE) return z;
    float t;
    return __fmul_rn(z, act_sigmoid(z, act, t));
}

// A pre-activation as the backward pass reads it: fp16 whatever the operands' type
// (three more bits than bf16 for the values it has: its rounding disappears
// behind that of dz), held at the largest fp16 value, beyond which every
// activation's slope is 0 or 1.  NaN stays NaN.
__device__ __forceinline__ __half preact_half(float z) {
    return __float2half_rn(z > 65504.0f ? 65504.0f : z < -65504.0f ? -65504.0f : z);
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

// Pairs of fp32 (packed arithmetic: half the instructions).
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

template <typename T, int G>
struct alignas(16) Group {
    T v[G];
};

// A group's elements as pairs of fp32, and back.
template <int G>
__device__ __forceinline__ void unpack(const Group<__nv_bfloat16, G>& g, float2 (&f)[G / 2]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(g.v);
#pragma unroll
    for (int i = 0; i < G / 2; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
template <int G>
__device__ __forceinline__ void unpack(const Group<__half, G>& g, float2 (&f)[G / 2]) {
    const __half2* w = reinterpret_cast<const __half2*>(g.v);
#pragma unroll
    for (int i = 0; i < G / 2; ++i) f[i] = __half22float2(w[i]);
}
template <int G>
__device__ __forceinline__ void unpack(const Group<float, G>& g, float2 (&f)[G / 2]) {
#pragma unroll
    for (int i = 0; i < G / 2; ++i) f[i] = make_float2(g.v[2 * i], g.v[2 * i + 1]);
}

// A group from shared memory in one 16-byte load (read through a reference it
// would be four 4-byte loads with four-way bank conflicts).
template <typename T, int G>
__device__ __forceinline__ Group<T, G> load_shared(const T* p) {
    Group<T, G> g;
    *reinterpret_cast<uint4*>(&g) = *reinterpret_cast<const uint4*>(p);
    return g;
}

template <typename T, int G>
__device__ __forceinline__ Group<T, G> pack(const float2 (&f)[G / 2]) {
    Group<T, G> g;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < G / 2; ++i) {
            g.v[2 * i] = f[i].x;
            g.v[2 * i + 1] = f[i].y;
        }
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < G / 2; ++i) reinterpret_cast<__half2*>(g.v)[i] = __floats2half2_rn(f[i].x, f[i].y);
    } else {
#pragma unroll
        for (int i = 0; i < G / 2; ++i) reinterpret_cast<__nv_bfloat162*>(g.v)[i] = __floats2bfloat162_rn(f[i].x, f[i].y);
    }
    return g;
}

// act(z) = z s and act'(z) = s + z s (1 - s) du/dz, u the sigmoid's argument, on a
// pair.
template <int ACT>
__device__ __forceinline__ void act_and_slope2(float2 z, float2& a, float2& slope) {
    if constexpr (ACT == Q6_ACT_NONE) {
        a = z;
        slope = both(1.0f);
    } else {
        float2 t, arg;
        if constexpr (ACT == Q6_ACT_GELU_TANH) {
            t = mul2(z, z);
            t = make_float2(fminf(t.x, 400.0f), fminf(t.y, 400.0f));
            arg = mul2(z, fma2(t, both(-kLog2e * kGelu2K * kGeluC), both(-kLog2e * kGelu2K)));
        } else {
            arg = mul2(z, both(-kLog2e));
        }
        const float2 d = add2(make_float2(ex2_f(arg.x), ex2_f(arg.y)), both(1.0f));
        const float2 s = make_float2(rcp_f(d.x), rcp_f(d.y));
        a = mul2(z, s);
        const float2 q = mul2(a, fma2(s, both(-1.0f), both(1.0f)));
        if constexpr (ACT == Q6_ACT_GELU_TANH)
            slope = fma2(q, fma2(t, both(3.0f * kGelu2K * kGeluC), both(kGelu2K)), s);
        else
            slope = add2(q, s);
    }
}

}  // namespace q6
