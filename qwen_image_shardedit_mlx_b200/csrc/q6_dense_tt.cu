// The dense product's kernels for both transposed (dz^T x).
#include "q6_dense_gemm.cuh"

namespace q6 {
Q6_DENSE_UNIT(tt, true, true)
}  // namespace q6
