// paged_attention_f32.cu -- paged attention over fp32 caches (paged_attention.cuh)
#include "paged_attention.cuh"

namespace tp {

int launch_paged_attention_f32(PagedAttentionArgs a, bool vec, cudaStream_t stream) {
  const int D = a.c.channels;
  int st;
  if (D <= 32) st = vec ? attend_by_group<float, 8, 1, true>(a, stream) : attend_by_group<float, 8, 1, false>(a, stream);
  else if (D <= 64) st = vec ? attend_by_group<float, 16, 1, true>(a, stream) : attend_by_group<float, 16, 1, false>(a, stream);
  else if (D <= 128) st = vec ? attend_by_group<float, 32, 1, true>(a, stream) : attend_by_group<float, 32, 1, false>(a, stream);
  else st = vec ? attend_by_group<float, 32, 2, true>(a, stream) : attend_by_group<float, 32, 2, false>(a, stream);
  return st != TP_OK ? st : join<float>(a, stream);
}

}  // namespace tp
