// residual_norm_f32_bwd.cu -- residual_norm.cu's backward for f32 rows.
#include "residual_norm.cuh"

namespace tp {

int launch_residual_norm_bwd_f32(int vec, int nv, const ResNormBwdArgs& g, size_t smem,
                                 int blocks, cudaStream_t s) {
#define RN_WARP(VEC, NV)                              \
  if (g.f.group == 32 && vec == VEC && nv == NV)       \
    return launch_bwd_known<float, VEC, NV, 32, RN_STAGED, false>(g, smem, blocks, s);
#define RN_BLOCK(VEC, NV)     \
  if (vec == VEC && nv == NV) \
    return launch_bwd_known<float, VEC, NV, 0, RN_F32, false>(g, smem, blocks, s);
  RN_WARP_F32(RN_WARP)
  RN_BLOCK_F32(RN_BLOCK)
#undef RN_WARP
#undef RN_BLOCK
  return TP_ERR_UNSUPPORTED;
}

}  // namespace tp
