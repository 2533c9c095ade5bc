// Matrix product of the dense linear, d = epilogue(Q P^T), in 16-bit operands
// with fp32 sums.  One CTA per 64 x 64 tile of d; 16 x 16 threads of 4 x 4
// outputs each; operand tiles of 16 along the sum are widened to fp32 in
// shared memory.
#include <algorithm>
#include <cstdint>

#include "q6_dense.cuh"
#include "q6_dense.h"
#include "q6_internal.h"
#include "q6_ptx.cuh"

namespace q6 {
namespace {

constexpr int kTile = 64, kStep = 16;

template <typename T>
__global__ void __launch_bounds__(256) dense_simple_kernel(DenseProduct a) {
    __shared__ float qs[kStep][kTile + 1], ps[kStep][kTile + 1];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t c0 = blockIdx.x * int64_t(kTile), r0 = blockIdx.y * int64_t(kTile);
    const int tc = threadIdx.x & 15, tr = threadIdx.x >> 4;
    const T* P = static_cast<const T*>(a.p);
    const T* Q = static_cast<const T*>(a.q);
    const int64_t pi = a.p_t ? 1 : a.ldp, pl = a.p_t ? a.ldp : 1, qi = a.q_t ? 1 : a.ldq, ql = a.q_t ? a.ldq : 1;
    float acc[4][4] = {};
    for (int64_t l0 = 0; l0 < a.L; l0 += kStep) {
        for (int e = threadIdx.x; e < kTile * kStep; e += 256) {
            const int i = e / kStep, l = e % kStep;
            qs[l][i] = r0 + i < a.R && l0 + l < a.L ? to_f(Q[(r0 + i) * qi + (l0 + l) * ql]) : 0.0f;
            ps[l][i] = c0 + i < a.C && l0 + l < a.L ? to_f(P[(c0 + i) * pi + (l0 + l) * pl]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int l = 0; l < kStep; ++l)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(qs[l][tr * 4 + i], ps[l][tc + 16 * j], acc[i][j]);
        __syncthreads();
    }
    const DenseEpilogue& e = a.epi;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t r = r0 + tr * 4 + i, c = c0 + tc + 16 * j;
            if (r >= a.R || c >= a.C) continue;
            float z = acc[i][j];
            if (e.bias) z += to_f(static_cast<const T*>(e.bias)[c]);
            if (e.preact) static_cast<T*>(e.preact)[r * a.C + c] = from_f<T>(z);
            float y = act_f(z, e.activation);
            if (e.gate) y *= to_f(static_cast<const T*>(e.gate)[r / e.rows_per_gate * e.ldg + c]);
            if (e.residual) y += to_f(static_cast<const T*>(e.residual)[r * e.ldr + c]);
            static_cast<T*>(a.d)[r * a.C + c] = from_f<T>(y);
        }
}

}  // namespace

size_t dense_product_workspace_bytes(int64_t, int64_t, int64_t, bool, bool) { return 0; }

int launch_dense_product(const DenseProduct& a, cudaStream_t stream) {
    const int64_t gx = (a.C + kTile - 1) / kTile, gy = (a.R + kTile - 1) / kTile;
    if (gy > 65535) return Q6_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
    const cudaError_t e =
        a.dtype == Q6_DTYPE_BF16
            ? launch_pdl(dense_simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, a)
            : launch_pdl(dense_simple_kernel<__half>, grid, dim3(256), 0, stream, a);
    return e == cudaSuccess ? Q6_OK : Q6_ERR_CUDA;
}

}  // namespace q6
