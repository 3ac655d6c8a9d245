// The low-rank adapter kernels for f16 operands (kernels: adapters_kernel.cuh).
#include "adapters_kernel.cuh"

namespace kairo {

KAIRO_LOW_RANK_LAUNCHES(__half)

}  // namespace kairo
