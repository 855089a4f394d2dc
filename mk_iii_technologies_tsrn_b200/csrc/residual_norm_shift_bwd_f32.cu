// residual_norm_shift_bwd_f32.cu -- residual_norm.cu's backward for fp32 rows that begin
// inside 16 bytes.
#include "residual_norm.cuh"

namespace tp {

int launch_residual_norm_bwd_shift_f32(int nv, const ResNormBwdArgs& g, size_t smem, int blocks,
                                       cudaStream_t s) {
#define RN_WARP(VEC, NV)           \
  if (g.f.group == 32 && nv == NV) \
    return launch_bwd_known<float, VEC, NV, 32, RN_STAGED, true>(g, smem, blocks, s);
  RN_SHIFT_WARP_F32(RN_WARP)
#undef RN_WARP
  return launch_bwd_known<float, 4, 2, 0, RN_STAGED, true>(g, smem, blocks, s);
}

}  // namespace tp
