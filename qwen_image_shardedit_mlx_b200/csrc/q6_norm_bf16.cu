// The layer norm's register kernels for bf16 rows.
#include "q6_norm.cuh"

namespace q6 {
Q6_NORM_TYPES(__nv_bfloat16, __nv_bfloat16)
Q6_NORM_TYPES(__nv_bfloat16, float)
Q6_NORM_UNIT(bf16)
}  // namespace q6
