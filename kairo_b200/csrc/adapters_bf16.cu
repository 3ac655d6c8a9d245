// The low-rank adapter kernels for bf16 operands (kernels: adapters_kernel.cuh).
#include "adapters_kernel.cuh"

namespace kairo {

KAIRO_LOW_RANK_LAUNCHES(__nv_bfloat16)

}  // namespace kairo
