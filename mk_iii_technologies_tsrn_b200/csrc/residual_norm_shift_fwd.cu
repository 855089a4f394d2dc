// residual_norm_shift_fwd.cu -- residual_norm.cu's forward for rows that begin inside
// 16 bytes.
#include "residual_norm.cuh"

namespace tp {

int launch_residual_norm_fwd_shift(int nv, const ResNormArgs& a, size_t smem, cudaStream_t s) {
#define RN_WARP(T, VEC, NV)                 \
  if (a.group == 32 && nv == NV)            \
    return launch_fwd_known<T, VEC, NV, 32, RN_STAGED, true>(a, smem, s);
#define RN_WARP_F(VEC, NV) RN_WARP(float, VEC, NV)
#define RN_WARP_B(VEC, NV) RN_WARP(bf16_t, VEC, NV)
  if (a.dtype == TP_DTYPE_BF16) {
    RN_SHIFT_WARP_BF16(RN_WARP_B)
    return launch_fwd_known<bf16_t, 8, 2, 0, RN_STAGED, true>(a, smem, s);
  }
  RN_SHIFT_WARP_F32(RN_WARP_F)
  return launch_fwd_known<float, 4, 2, 0, RN_STAGED, true>(a, smem, s);
#undef RN_WARP_B
#undef RN_WARP_F
#undef RN_WARP
}

}  // namespace tp
