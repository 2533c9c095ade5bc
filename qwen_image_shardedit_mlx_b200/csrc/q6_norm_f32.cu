// The layer norm's register kernels for fp32 rows.
#include "q6_norm.cuh"

namespace q6 {
Q6_NORM_TYPES(float, float)
Q6_NORM_UNIT(f32)
}  // namespace q6
