// capi_decode.cu -- the extern "C" boundary of the decoding operators: validation on the
// host, then the launches (as capi.cu does for the others).
#include "decode.cuh"

using namespace tp;

namespace {

cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
bool is_float_code(int dtype) { return dtype == TP_DTYPE_F32 || dtype == TP_DTYPE_BF16; }

// `rows`: whether any sequence looks into the cache
int paged_cache(PagedCache& c, int dtype, const tp_paged_cache* p, bool rows) {
  TP_RETURN_IF(!is_float_code(dtype), TP_ERR_UNSUPPORTED);
  TP_RETURN_IF(p == nullptr, TP_ERR_NULL_POINTER);
  TP_RETURN_IF(p->pages < 0 || p->page_size < 1 || p->heads < 0 || p->channels < 0 ||
                   p->table_cols < 0 || p->table_row < 0,
               TP_ERR_INVALID_ARG);
  for (int64_t s : {p->k_page, p->k_slot, p->k_head, p->v_page, p->v_slot, p->v_head})
    TP_RETURN_IF(s < 0, TP_ERR_INVALID_ARG);
  // (slots are counted in 32 bits; tiles look a few past the end)
  TP_RETURN_IF(p->page_size > INT32_MAX || p->table_cols > INT32_MAX || p->heads > INT32_MAX ||
                   p->channels > INT32_MAX / 16 ||
                   (p->channels > 0 && p->heads > INT32_MAX / 16 / p->channels) ||
                   (p->table_cols > 0 && p->page_size > ((int64_t)INT32_MAX - 65536) / p->table_cols),
               TP_ERR_TOO_LARGE);
  if (rows && p->table_cols > 0) {
    TP_CHECK_PTR(p->table);
    if (p->pages > 0 && p->heads > 0 && p->channels > 0) {
      TP_CHECK_PTR(p->k);
      TP_CHECK_PTR(p->v);
    }
  }
  const int64_t e = dtype == TP_DTYPE_BF16 ? 2 : 4;
  c.k = (char*)p->k;
  c.v = (char*)p->v;
  c.pages = p->pages;
  c.page_size = (int)p->page_size;
  c.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (c.page_size == 1 << i) c.page_shift = i;
  c.heads = (int)p->heads;
  c.channels = (int)p->channels;
  c.esize = (int)e;
  c.k_page = p->k_page * e;
  c.k_slot = p->k_slot * e;
  c.k_head = p->k_head * e;
  c.v_page = p->v_page * e;
  c.v_slot = p->v_slot * e;
  c.v_head = p->v_head * e;
  c.table = p->table;
  c.table_row = p->table_row;
  c.table_cols = (int)p->table_cols;
  return TP_OK;
}

bool attention_sizes(int64_t B, int64_t H, int64_t heads, int64_t channels) {
  return B >= 0 && H >= 0 && heads >= 1 && H % heads == 0 && channels >= 1;
}

}  // namespace

extern "C" {

int64_t tp_paged_attention_workspace_bytes(int dtype, int64_t B, int64_t H, int64_t heads,
                                           int64_t channels, int64_t slots, int mass) {
  if (!is_float_code(dtype) || !attention_sizes(B, H, heads, channels) || slots < 0 ||
      slots > INT32_MAX)
    return -1;
  if (B == 0 || H == 0) return 0;
  return paged_attention_cut(B, H, heads, channels, slots, mass != 0).bytes();
}

int tp_paged_attention(int dtype, int64_t B, int64_t H, const tp_paged_cache* cache,
                       const int32_t* lengths, const void* q, int64_t q_sb, int64_t q_sh,
                       const void* key, int64_t key_sb, int64_t key_sh, const void* value,
                       int64_t value_sb, int64_t value_sh, const float* gate, const float* tau,
                       float scale, float* mass, int64_t mass_sb, int64_t mass_sh,
                       int64_t mass_slots, void* out, void* workspace, int64_t workspace_bytes,
                       void* stream) {
  PagedAttentionArgs a{};
  const int st = paged_cache(a.c, dtype, cache, B > 0 && H > 0);
  if (st != TP_OK) return st;
  TP_RETURN_IF(!attention_sizes(B, H, cache->heads, cache->channels), TP_ERR_INVALID_ARG);
  TP_RETURN_IF(cache->channels > 256, TP_ERR_UNSUPPORTED);
  TP_RETURN_IF(q_sb < 0 || q_sh < 0 || (key == nullptr) != (value == nullptr), TP_ERR_INVALID_ARG);
  if (key != nullptr)
    TP_RETURN_IF(key_sb < 0 || key_sh < 0 || value_sb < 0 || value_sh < 0, TP_ERR_INVALID_ARG);
  if (mass != nullptr)
    TP_RETURN_IF(mass_sb < 0 || mass_sh < 0 || mass_slots < 0, TP_ERR_INVALID_ARG);
  if (B == 0 || H == 0) return TP_OK;
  int64_t capacity = cache->table_cols * cache->page_size;
  if (mass != nullptr && mass_slots < capacity) capacity = mass_slots;
  const PagedAttentionCut cut = paged_attention_cut(B, H, cache->heads, cache->channels,
                                                    capacity, mass != nullptr);
  TP_RETURN_IF(B > INT32_MAX || H > INT32_MAX || B * H > INT32_MAX / 16 ||
                   B * cache->heads > (INT32_MAX - B * H) / (capacity / MASS_SLOTS + 1),
               TP_ERR_TOO_LARGE);
  TP_CHECK_PTR(lengths);
  TP_CHECK_PTR(q);
  TP_CHECK_PTR(out);
  for (const void* p : {key, value, (const void*)gate, (const void*)tau, (const void*)mass})
    TP_CHECK_OPT_PTR(p);
  TP_RETURN_IF(workspace == nullptr || workspace_bytes < cut.bytes(), TP_ERR_WORKSPACE);
  TP_CHECK_PTR(workspace);
  TP_RETURN_IF(!aligned16(workspace), TP_ERR_MISALIGNED);
  a.dtype = dtype;
  a.B = (int)B;
  a.H = (int)H;
  a.group = (int)(H / cache->heads);
  a.capacity = (int)capacity;
  a.q = q;
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.lengths = lengths;
  a.key = key;
  a.value = value;
  a.key_sb = key_sb;
  a.key_sh = key_sh;
  a.value_sb = value_sb;
  a.value_sh = value_sh;
  a.gate = gate;
  a.tau = tau;
  a.scale = scale;
  a.mass = mass;
  a.mass_sb = mass_sb;
  a.mass_sh = mass_sh;
  a.out = out;
  float* ws = (float*)workspace;
  a.scores = mass != nullptr ? ws : nullptr;
  a.score_row = cut.score_row;
  a.runs_of = (int2*)(ws + cut.scores);
  a.ml = (float2*)(ws + cut.scores + cut.runs);
  a.part = ws + cut.scores + cut.runs + cut.ml;
  a.bad = index_error_words();
  return launch_paged_attention(a, as_stream(stream));
}

int tp_paged_append(int dtype, int64_t B, int64_t T, const tp_paged_cache* cache,
                    const int32_t* starts, const int32_t* counts, const void* key, int64_t key_sb,
                    int64_t key_st, int64_t key_sh, const void* value, int64_t value_sb,
                    int64_t value_st, int64_t value_sh, void* stream) {
  PagedAppendArgs a{};
  const int st = paged_cache(a.c, dtype, cache, B > 0 && T > 0);
  if (st != TP_OK) return st;
  TP_RETURN_IF(B < 0 || T < 0, TP_ERR_INVALID_ARG);
  for (int64_t s : {key_sb, key_st, key_sh, value_sb, value_st, value_sh})
    TP_RETURN_IF(s < 0, TP_ERR_INVALID_ARG);
  if (B == 0 || T == 0 || cache->heads == 0 || cache->channels == 0) return TP_OK;
  TP_RETURN_IF(T > INT32_MAX || B > INT32_MAX ||
                   cache->heads * cache->channels > INT64_MAX / 8 / (B * T),
               TP_ERR_TOO_LARGE);
  TP_CHECK_PTR(starts);
  TP_CHECK_OPT_PTR(counts);
  TP_CHECK_PTR(key);
  TP_CHECK_PTR(value);
  const int64_t e = a.c.esize;
  a.B = B;
  a.T = T;
  a.key = (const char*)key;
  a.value = (const char*)value;
  a.key_sb = key_sb * e;
  a.key_st = key_st * e;
  a.key_sh = key_sh * e;
  a.value_sb = value_sb * e;
  a.value_st = value_st * e;
  a.value_sh = value_sh * e;
  a.starts = starts;
  a.counts = counts;
  a.bad = index_error_words();
  return launch_paged_append(a, as_stream(stream));
}

int tp_cache_evict(int dtype, int64_t B, const tp_paged_cache* cache, const int32_t* lengths,
                   const float* mass, int64_t mass_sb, int64_t mass_sh, int64_t mass_slots,
                   float* out, int64_t out_sb, int64_t out_sh, int64_t keep, int64_t recent,
                   int32_t* kept, void* stream) {
  CacheEvictArgs a{};
  const int st = paged_cache(a.c, dtype, cache, B > 0);
  if (st != TP_OK) return st;
  TP_RETURN_IF(B < 0 || keep < 1 || recent < 0 || recent > keep || mass_slots < 0 || mass_sb < 0 ||
                   mass_sh < 0 || out_sb < 0 || out_sh < 0,
               TP_ERR_INVALID_ARG);
  if (B == 0 || cache->heads == 0) return TP_OK;
  int64_t capacity = cache->table_cols * cache->page_size;
  if (mass_slots < capacity) capacity = mass_slots;
  TP_RETURN_IF(keep > (int64_t)INT32_MAX - 65536 || B > INT32_MAX ||
                   B * cache->heads > INT32_MAX / (2 * (cache->channels + 1)),
               TP_ERR_TOO_LARGE);
  TP_CHECK_PTR(lengths);
  TP_CHECK_PTR(mass);
  TP_CHECK_PTR(out);
  TP_CHECK_PTR(kept);
  a.B = B;
  a.capacity = (int)capacity;
  a.lengths = lengths;
  a.mass = mass;
  a.mass_sb = mass_sb;
  a.mass_sh = mass_sh;
  a.out = out;
  a.out_sb = out_sb;
  a.out_sh = out_sh;
  a.keep = (int)keep;
  a.recent = (int)recent;
  a.kept = kept;
  a.bad = index_error_words();
  return launch_cache_evict(a, as_stream(stream));
}

int tp_sample_tokens(int dtype, int64_t B, int64_t V, const void* logits, int64_t ld,
                     int uniform_bits, const void* uniform, double temperature,
                     const float* temperatures, int64_t top_k, const int32_t* top_ks, double top_p,
                     const float* top_ps, double min_p, const float* min_ps, int64_t* token,
                     float* logprob, void* stream) {
  TP_RETURN_IF(B < 0 || V < 1 || ld < 0 || (uniform_bits != 32 && uniform_bits != 64),
               TP_ERR_INVALID_ARG);
  TP_RETURN_IF(!is_float_code(dtype), TP_ERR_UNSUPPORTED);
  TP_RETURN_IF(V >= SAMPLE_MAX_TOKENS || B > INT32_MAX / 8, TP_ERR_TOO_LARGE);
  if (B == 0) return TP_OK;
  TP_CHECK_PTR(logits);
  TP_CHECK_PTR(uniform);
  TP_CHECK_PTR(token);
  for (const void* p : {(const void*)temperatures, (const void*)top_ks, (const void*)top_ps,
                        (const void*)min_ps, (const void*)logprob})
    TP_CHECK_OPT_PTR(p);
  SampleArgs a{};
  a.dtype = dtype;
  a.B = B;
  a.V = V;
  a.ld = ld;
  a.logits = logits;
  a.uniform = uniform;
  a.uniform64 = uniform_bits == 64;
  a.temperature = {temperatures, temperature};
  a.top_p = {top_ps, top_p};
  a.min_p = {min_ps, min_p};
  a.top_k_of_row = top_ks;
  a.top_k = top_k;
  a.token = token;
  a.logprob = logprob;
  return launch_sample_tokens(a, as_stream(stream));
}

}  // extern "C"
