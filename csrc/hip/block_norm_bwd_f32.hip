// Backward of the gated residual norm, float32.
#include <hip/hip_runtime.h>

#include "block_norm_bwd.h"

namespace pbx {
void launch_residual_bwd_f32(const ResidualArgs& a, int grid, hipStream_t s) { residual_bwd<kF32, kF32>(a, grid, s); }
}  // namespace pbx
