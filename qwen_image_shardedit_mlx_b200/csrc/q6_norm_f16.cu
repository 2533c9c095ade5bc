// The layer norm's register kernels for fp16 rows.
#include "q6_norm.cuh"

namespace q6 {
Q6_NORM_TYPES(__half, __half)
Q6_NORM_TYPES(__half, float)
Q6_NORM_UNIT(f16)
}  // namespace q6
