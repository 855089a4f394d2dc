// decode.cuh -- argument structs and launchers of the decoding operators: attention of
// one new token over a paged key-value cache, writing a prompt into it, eviction from
// it, and sampling of the next token.
#pragma once

#include "common.cuh"

namespace tp {

// A cache of pages (tp_paged_cache) with its strides in BYTES.
struct PagedCache {
  char* k;
  char* v;
  int64_t pages;
  int page_size, page_shift, heads, channels, esize;      // page_shift: -1 if no power of two
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  const int* table;
  int64_t table_row;       // elements from one sequence's row to the next
  int table_cols;
  // the column of a slot's page in its sequence's row, and its place in the page
  __device__ __forceinline__ int column(int slot) const {
    return page_shift >= 0 ? slot >> page_shift : slot / page_size;
  }
  __device__ __forceinline__ int within(int slot, int column) const { return slot - column * page_size; }
};

struct PagedAttentionArgs {
  PagedCache c;
  int dtype;
  int B, H, group;         // group: query heads of a key head
  int capacity;            // slots a sequence may use
  const void* q;
  int64_t q_sb, q_sh;      // elements
  const int* lengths;
  const void* key;         // the new token's, or NULL
  const void* value;
  int64_t key_sb, key_sh, value_sb, value_sh;
  const float* gate;       // [B, H], or NULL
  const float* tau;        // [H], or NULL
  float scale;
  float* mass;             // [B, heads, slots], or NULL
  int64_t mass_sb, mass_sh;
  void* out;               // [B, H, channels]
  // the split of the work (paged_attention.cuh), chosen with the kernel
  int block_heads;         // query heads that a warp takes at a time
  int head_blocks;         // blocks of them over a key head
  int runs, tile;          // runs of the list of tiles, slots of a tile
  int2* runs_of;           // [B] the first run with a segment of the sequence, and how many have
  float2* ml;              // [segments][block_heads] (maximum, sum) of a segment, base 2
  float* part;             // [segments][block_heads][channels] sums of a segment
  float* scores;           // [B * H][score_row] scores, base 2, where mass is wanted
  int64_t score_row;       // a multiple of four
  IndexErrorWords bad;
};

constexpr int MASS_SLOTS = 1024;     // slots that a block adds weights to

constexpr int ATT_WARPS = 4;         // of a block
constexpr int ATT_MOST_BLOCKS = 4;   // on an SM

struct PagedAttentionCut {
  int64_t scores, runs, ml, part, score_row;      // floats, in this order in the workspace
  int64_t bytes() const { return 4 * (scores + runs + ml + part); }
};
PagedAttentionCut paged_attention_cut(int64_t B, int64_t H, int64_t heads, int64_t D,
                                      int64_t capacity, bool mass);
int launch_paged_attention(PagedAttentionArgs a, cudaStream_t stream);
// vec: rows of the cache, the key and the value begin and end on 16 bytes
int launch_paged_attention_f32(PagedAttentionArgs a, bool vec, cudaStream_t stream);
int launch_paged_attention_bf16(PagedAttentionArgs a, bool vec, cudaStream_t stream);

struct PagedAppendArgs {
  PagedCache c;
  int64_t B, T;
  const char* key;
  const char* value;
  int64_t key_sb, key_st, key_sh, value_sb, value_st, value_sh;     // bytes
  const int* starts;
  const int* counts;             // or NULL: T
  IndexErrorWords bad;
};
int launch_paged_append(const PagedAppendArgs& a, cudaStream_t stream);

struct CacheEvictArgs {
  PagedCache c;
  int64_t B;
  int capacity;
  const int* lengths;
  const float* mass;
  int64_t mass_sb, mass_sh;
  float* out;                    // mass of the kept slots; may be `mass`
  int64_t out_sb, out_sh;
  int keep, recent;
  int* kept;                     // [B, heads, keep]
  IndexErrorWords bad;
};
int launch_cache_evict(const CacheEvictArgs& a, cudaStream_t stream);

// one choice for all rows, or one of each
struct RowChoice {
  const float* of_row;           // NULL: `all`
  double all;
};
struct SampleArgs {
  int dtype;
  int64_t B, V, ld;
  const void* logits;
  const void* uniform;           // [B]
  int uniform64;
  RowChoice temperature, top_p, min_p;
  const int* top_k_of_row;       // NULL: top_k
  int64_t top_k;
  int64_t* token;                // [B]
  float* logprob;                // [B], or NULL
};
constexpr int64_t SAMPLE_MAX_TOKENS = 1 << 19;
int launch_sample_tokens(const SampleArgs& a, cudaStream_t stream);

}  // namespace tp
