// Backward of the gated residual norm, bfloat16 on a float32 stream.
#include <hip/hip_runtime.h>

#include "block_norm_bwd.h"

namespace pbx {
void launch_residual_bwd_f32_bf16(const ResidualArgs& a, int grid, hipStream_t s) { residual_bwd<kF32, kBF16>(a, grid, s); }
}  // namespace pbx
