// residual_norm_shift_bwd_bf16.cu -- residual_norm.cu's backward for bf16 rows that begin
// inside 16 bytes.
#include "residual_norm.cuh"

namespace tp {

int launch_residual_norm_bwd_shift_bf16(int nv, const ResNormBwdArgs& g, size_t smem, int blocks,
                                       cudaStream_t s) {
#define RN_WARP(VEC, NV)           \
  if (g.f.group == 32 && nv == NV) \
    return launch_bwd_known<bf16_t, VEC, NV, 32, RN_STAGED, true>(g, smem, blocks, s);
  RN_SHIFT_WARP_BF16(RN_WARP)
#undef RN_WARP
  return launch_bwd_known<bf16_t, 8, 2, 0, RN_STAGED, true>(g, smem, blocks, s);
}

}  // namespace tp
