// Backward of the gated residual norm, float16.
#include <hip/hip_runtime.h>

#include "block_norm_bwd.h"

namespace pbx {
void launch_residual_bwd_f16(const ResidualArgs& a, int grid, hipStream_t s) { residual_bwd<kF16, kF16>(a, grid, s); }
}  // namespace pbx
