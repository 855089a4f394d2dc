// residual_norm_f32_fwd.cu -- residual_norm.cu's forward for f32 rows.
#include "residual_norm.cuh"

namespace tp {

int launch_residual_norm_fwd_f32(int vec, int nv, const ResNormArgs& a, size_t smem,
                                 cudaStream_t s) {
#define RN_WARP(VEC, NV)                              \
  if (a.group == 32 && vec == VEC && nv == NV)       \
    return launch_fwd_known<float, VEC, NV, 32, RN_STAGED, false>(a, smem, s);
#define RN_BLOCK(VEC, NV)     \
  if (vec == VEC && nv == NV) \
    return launch_fwd_known<float, VEC, NV, 0, RN_F32, false>(a, smem, s);
  RN_WARP_F32(RN_WARP)
  RN_BLOCK_F32(RN_BLOCK)
#undef RN_WARP
#undef RN_BLOCK
  return TP_ERR_UNSUPPORTED;
}

}  // namespace tp
