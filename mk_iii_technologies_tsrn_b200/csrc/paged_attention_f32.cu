// paged_attention_f32.cu -- paged attention over fp32 caches (paged_attention.cuh)
#include "paged_attention.cuh"

namespace tp {

namespace {

// One query head at a time, two, or four: registers hold no more of their channels and sums.
template <int LPK, int NCH>
int by_group(PagedAttentionArgs& a, bool vec, cudaStream_t stream) {
  const bool gated = a.gate != nullptr;
  if (!vec)
    return gated ? attend<float, LPK, NCH, 1, true, false>(a, stream)
                 : attend<float, LPK, NCH, 1, false, false>(a, stream);
  if (a.group == 1)
    return gated ? attend<float, LPK, NCH, 1, true, true>(a, stream)
                 : attend<float, LPK, NCH, 1, false, true>(a, stream);
  if (a.group == 2)
    return gated ? attend<float, LPK, NCH, 2, true, true>(a, stream)
                 : attend<float, LPK, NCH, 2, false, true>(a, stream);
  return gated ? attend<float, LPK, NCH, 4, true, true>(a, stream)
               : attend<float, LPK, NCH, 4, false, true>(a, stream);
}

}  // namespace

int launch_paged_attention_f32(PagedAttentionArgs a, bool vec, cudaStream_t stream) {
  const int D = a.c.channels;
  return D <= 32    ? by_group<8, 1>(a, vec, stream)
         : D <= 64  ? by_group<16, 1>(a, vec, stream)
         : D <= 128 ? by_group<32, 1>(a, vec, stream)
                    : by_group<32, 2>(a, vec, stream);
}

}  // namespace tp
