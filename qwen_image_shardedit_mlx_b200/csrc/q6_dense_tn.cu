// The dense product's kernels for P transposed (dz W).
#include "q6_dense_gemm.cuh"

namespace q6 {
Q6_DENSE_UNIT(tn, true, false)
}  // namespace q6
