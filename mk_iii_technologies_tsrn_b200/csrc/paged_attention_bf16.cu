// paged_attention_bf16.cu -- paged attention over bf16 caches (paged_attention.cuh)
#include "paged_attention.cuh"

namespace tp {

int launch_paged_attention_bf16(PagedAttentionArgs a, bool vec, cudaStream_t stream) {
  const int D = a.c.channels;
  int st;
  if (D <= 64) st = vec ? attend_by_group<uint16_t, 8, 1, true>(a, stream) : attend_by_group<uint16_t, 8, 1, false>(a, stream);
  else if (D <= 128) st = vec ? attend_by_group<uint16_t, 16, 1, true>(a, stream) : attend_by_group<uint16_t, 16, 1, false>(a, stream);
  else st = vec ? attend_by_group<uint16_t, 32, 1, true>(a, stream) : attend_by_group<uint16_t, 32, 1, false>(a, stream);
  return st != TP_OK ? st : join<uint16_t>(a, stream);
}

}  // namespace tp
