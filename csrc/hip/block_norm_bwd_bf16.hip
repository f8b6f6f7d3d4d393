// Backward of the gated residual norm, bfloat16.
#include <hip/hip_runtime.h>

#include "block_norm_bwd.h"

namespace pbx {
void launch_residual_bwd_bf16(const ResidualArgs& a, int grid, hipStream_t s) { residual_bwd<kBF16, kBF16>(a, grid, s); }
}  // namespace pbx
