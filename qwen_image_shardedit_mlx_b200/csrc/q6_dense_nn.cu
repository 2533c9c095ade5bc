// The dense product's kernels for both operands with the sum contiguous (x W^T).
#include "q6_dense_gemm.cuh"

namespace q6 {
Q6_DENSE_UNIT(nn, false, false)
}  // namespace q6
