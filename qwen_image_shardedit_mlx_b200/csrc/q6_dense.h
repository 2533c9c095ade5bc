// Host-side interfaces between the dense linear's entry points (q6_dense.cu)
// and its matrix products (q6_dense_gemm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "q6_b200.h"

namespace q6 {

// Epilogue of a product: d = residual + gate * act(sum + bias), preact = sum + bias.
// Every pointer may be null.  Vectors and matrices are in the product's dtype.
struct DenseEpilogue {
    const void* bias = nullptr;      // [C]
    const void* gate = nullptr;      // [R / rows_per_gate, C], ldg elements apart
    int64_t ldg = 0, rows_per_gate = 1;
    const void* residual = nullptr;  // [R, C], row stride ldr
    int64_t ldr = 0;
    void* preact = nullptr;          // [R, C] dense, fp16 (preact_half) or (preact_f32) fp32
    bool preact_f32 = false;
    int activation = Q6_ACT_NONE;
};

// d[r, c] = epilogue(sum_l Q(r, l) P(c, l)),  r < R, c < C, l < L; d dense [R, C].
// An operand is stored [index][l] (its l contiguous) or, with the _t flag,
// transposed: [l][index]; ld* is the stride between stored rows.
struct DenseProduct {
    const void* p;
    int64_t ldp;
    bool p_t;
    const void* q;
    int64_t ldq;
    bool q_t;
    void* d;
    int64_t R, C, L;
    int dtype;  // Q6_DTYPE_BF16 or Q6_DTYPE_F16
    DenseEpilogue epi;
    void* workspace = nullptr;  // dense_product_workspace_bytes(...) bytes
    size_t workspace_bytes = 0;
};

// A few rows of Q (R <= 16), both operands with the sum contiguous, any alignment,
// no workspace (q6_dense_rows.cu).
bool dense_few_rows(int64_t R, int64_t C, int64_t L);  // where it is the faster path
int launch_dense_rows(const DenseProduct& a, cudaStream_t stream);

int launch_dense_product(const DenseProduct& a, cudaStream_t stream);
size_t dense_product_workspace_bytes(int64_t R, int64_t C, int64_t L, bool p_t, bool q_t);

}  // namespace q6
