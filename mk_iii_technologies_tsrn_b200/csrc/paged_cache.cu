// paged_cache.cu -- what surrounds paged attention: the split of its rows, writing of
// prompts into the pages, and eviction from them by accumulated attention weight.
#include <algorithm>

#include "decode.cuh"

namespace tp {

PagedAttentionCut paged_attention_cut(int64_t B, int64_t H, int64_t heads, int64_t D,
                                      int64_t capacity, bool mass) {
  // one for each sequence and each run, for every query head, their number rounded up to blocks
  // of at most eight of a key head
  const int64_t heads8 = heads * (H / heads + 7);
  const int64_t segments = B * heads8 + std::max(heads8, 8 * (int64_t)num_sms() * ATT_WARPS * ATT_MOST_BLOCKS);
  PagedAttentionCut cut{};
  cut.score_row = ceil_div(capacity, 4) * 4;
  if (mass) cut.scores = B * H * cut.score_row;
  cut.runs = ceil_div(B, 2) * 4;
  cut.ml = ceil_div(segments, 2) * 4;
  cut.part = segments * D;
  return cut;
}

namespace {
bool rows16(const void* p, int64_t s0, int64_t s1, int64_t s2) {
  return aligned16(p) && ((s0 | s1 | s2) & 15) == 0;
}
}  // namespace

int launch_paged_attention(PagedAttentionArgs a, cudaStream_t stream) {
  const PagedCache& c = a.c;
  const int e = c.esize;
  const bool vec = (c.channels * e) % 16 == 0 && rows16(c.k, c.k_page, c.k_slot, c.k_head) &&
                   rows16(c.v, c.v_page, c.v_slot, c.v_head) &&
                   (a.key == nullptr || (rows16(a.key, a.key_sb * e, a.key_sh * e, 0) &&
                                         rows16(a.value, a.value_sb * e, a.value_sh * e, 0)));
  return a.dtype == TP_DTYPE_BF16 ? launch_paged_attention_bf16(a, vec, stream)
                                  : launch_paged_attention_f32(a, vec, stream);
}

namespace {

// ---------------------------------------------------------------- append
// A warp's lanes go along the words of (token, head) rows; one word of key and value each.
// W: bytes of a word that every row's begin, stride and length are multiples of.
template <typename W>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppendArgs a, int words) {
  const int64_t per_token = (int64_t)a.c.heads * words, total = a.B * a.T * per_token;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t token = i / per_token;
    const int rest = (int)(i - token * per_token), head = rest / words, w = rest - head * words;
    const int64_t b = token / a.T, t = token - b * a.T;
    if (a.counts != nullptr && t >= __ldg(a.counts + b)) continue;
    const int64_t slot = (int64_t)__ldg(a.starts + b) + t;
    const int64_t col = slot / a.c.page_size;
    int page = -1;
    if (slot >= 0 && col < a.c.table_cols) page = __ldg(a.c.table + b * a.c.table_row + col);
    if (page < 0 || page >= a.c.pages) {
      tp_record_index_error(a.bad.error, a.bad.seen);
      continue;
    }
    const int64_t in = slot - col * a.c.page_size;
    const W k = __ldg((const W*)(a.key + b * a.key_sb + t * a.key_st + head * a.key_sh) + w);
    const W v = __ldg((const W*)(a.value + b * a.value_sb + t * a.value_st + head * a.value_sh) + w);
    *((W*)(a.c.k + page * a.c.k_page + in * a.c.k_slot + head * a.c.k_head) + w) = k;
    *((W*)(a.c.v + page * a.c.v_page + in * a.c.v_slot + head * a.c.v_head) + w) = v;
  }
}

template <typename W>
int append(const PagedAppendArgs& a, cudaStream_t stream) {
  const int words = a.c.channels * a.c.esize / (int)sizeof(W);
  const int64_t total = a.B * a.T * a.c.heads * words;
  const int64_t blocks = std::min<int64_t>(ceil_div(total, 256), (int64_t)num_sms() * 32);
  paged_append_kernel<W><<<(unsigned)blocks, 256, 0, stream>>>(a, words);
  return launch_status();
}

// ---------------------------------------------------------------- evict
__device__ __forceinline__ uint32_t ordered_bits(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);          // (-0 is 0)
  return f != f ? 0xffffffffu : (u & 0x80000000u ? ~u : u | 0x80000000u);
}

// One block per sequence and key head: the kept slots, in order, and their mass.
constexpr int EVICT_THREADS = 1024;

// exclusive sum over the block of each thread's v; `total` gets the sum
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_sums[32 + lane] = s;
  }
  __syncthreads();
  const int before = warp ? warp_sums[32 + warp - 1] : 0;
  total = warp_sums[63];
  __syncthreads();
  return before + x - v;
}

__global__ void __launch_bounds__(EVICT_THREADS) evict_select_kernel(const CacheEvictArgs a) {
  __shared__ int hist[256];
  __shared__ int sums[64];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int kvh = blockIdx.x % a.c.heads, b = blockIdx.x / a.c.heads, tid = threadIdx.x;
  const int given = __ldg(a.lengths + b);
  const bool bad = given < 0 || given > a.capacity;
  if (bad && tid == 0) tp_record_index_error(a.bad.error, a.bad.seen);
  const int n = bad ? 0 : given;
  const float* mass = a.mass + (int64_t)b * a.mass_sb + (int64_t)kvh * a.mass_sh;
  float* out = a.out + (int64_t)b * a.out_sb + (int64_t)kvh * a.out_sh;
  int* kept = a.kept + (int64_t)blockIdx.x * a.keep;
  if (n <= a.keep) {
    for (int i = tid; i < a.keep; i += EVICT_THREADS) {
      kept[i] = i < n ? i : -1;
      if (i < n && out != mass) out[i] = mass[i];
    }
    return;
  }
  // slots before `old` compete for `need` places
  const int old = n - min(a.recent, n), need = a.keep - (n - old);
  uint32_t prefix = 0;
  int left = need;                 // places among the slots whose high bits are `prefix`
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < old; i += EVICT_THREADS) {
        const uint32_t u = ordered_bits(mass[i]);
        if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid < 32) {              // the digit where the sum from above passes `left`
        int mine[8], all = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) all += mine[k] = hist[255 - (tid * 8 + k)];
        int above = all;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int y = __shfl_up_sync(0xffffffffu, above, o);
          if (tid >= o) above += y;
        }
        above -= all;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (above < left && above + mine[k] >= left) {
            s_prefix = prefix | (uint32_t)(255 - (tid * 8 + k)) << shift;
            s_need = left - above;
          }
          above += mine[k];
        }
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_need;
      __syncthreads();
    }
  }
  // in order of the slots: those above `prefix`, the first `left` of those equal to it, and
  // the recent ones
  int taken = 0, ties = 0;
  for (int base = 0; base < n; base += EVICT_THREADS) {
    const int i = base + tid;
    const float m = i < n ? mass[i] : 0.0f;
    const uint32_t u = ordered_bits(m);
    const bool tie = need > 0 && i < old && u == prefix;
    int all;
    const int rank = block_scan(tie, sums, all);
    const bool take = i < n && (i >= old || (need > 0 && (u > prefix || (tie && ties + rank < left))));
    ties += all;
    const int at = taken + block_scan(take, sums, all);
    taken += all;
    // (at <= i, and every slot of this step has been read: `out` may be `mass`)
    if (take) {
      kept[at] = i;
      out[at] = m;
    }
  }
}

// Moves kept rows to the front.  Different words of a row move apart from one another: a
// block takes one or more words of all kept rows of a sequence and head, in order.  Row i
// comes from kept[i] >= i, so a step's rows are read before any of them is written, and no
// later step reads what an earlier one wrote.
constexpr int MOVE_THREADS = 256, MOVE_DEPTH = 8;
template <typename W>
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const CacheEvictArgs a, int words,
                                                                  int width, int slices) {
  int r = blockIdx.x;
  const int slice = r % slices;
  r /= slices;
  const bool value = r % 2;
  r /= 2;
  const int kvh = r % a.c.heads, b = r / a.c.heads;
  const int n = __ldg(a.lengths + b);
  if (n < 0 || n > a.capacity || n <= a.keep) return;
  const int* kept = a.kept + (int64_t)r * a.keep;
  const int* row = a.c.table + (int64_t)b * a.c.table_row;
  char* const base = value ? a.c.v + kvh * a.c.v_head : a.c.k + kvh * a.c.k_head;
  const int64_t page_bytes = value ? a.c.v_page : a.c.k_page, slot_bytes = value ? a.c.v_slot : a.c.k_slot;
  const int w = slice * width + threadIdx.x % width;
  const int per = MOVE_THREADS / width, first = threadIdx.x / width;
  auto at = [&](int slot) -> W* {
    const int page = __ldg(row + slot / a.c.page_size);
    if (page < 0 || page >= a.c.pages) {
      tp_record_index_error(a.bad.error, a.bad.seen);
      return nullptr;
    }
    return (W*)(base + (int64_t)page * page_bytes + (int64_t)(slot % a.c.page_size) * slot_bytes) + w;
  };
  for (int i0 = 0; i0 < a.keep; i0 += per * MOVE_DEPTH) {
    W x[MOVE_DEPTH];
    W* to[MOVE_DEPTH];
#pragma unroll
    for (int k = 0; k < MOVE_DEPTH; ++k) {
      const int i = i0 + k * per + first;
      to[k] = nullptr;
      if (first < per && i < a.keep && w < words) {
        const int from = __ldg(kept + i);
        if (from != i) {
          const W* src = at(from);
          if (src != nullptr) {
            to[k] = at(i);
            x[k] = *src;
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < MOVE_DEPTH; ++k)
      if (to[k] != nullptr) *to[k] = x[k];
  }
}

template <typename W>
int move(const CacheEvictArgs& a, cudaStream_t stream) {
  const int words = a.c.channels * a.c.esize / (int)sizeof(W);
  const int width = std::min(words, std::max(1, 64 / (int)sizeof(W)));
  const int slices = (words + width - 1) / width;
  const int64_t blocks = a.B * a.c.heads * 2 * slices;
  TP_RETURN_IF(blocks > INT32_MAX, TP_ERR_TOO_LARGE);
  evict_move_kernel<W><<<(unsigned)blocks, MOVE_THREADS, 0, stream>>>(a, words, width, slices);
  return launch_status();
}

// the widest word (16, 8, 4 or 2 bytes) that divides all of them
int word_bytes(std::initializer_list<int64_t> of) {
  int64_t all = 0;
  for (int64_t x : of) all |= x;
  return (all & 15) == 0 ? 16 : (all & 7) == 0 ? 8 : (all & 3) == 0 ? 4 : 2;
}
int64_t address(const void* p) { return (int64_t)(uintptr_t)p; }

}  // namespace

int launch_paged_append(const PagedAppendArgs& a, cudaStream_t stream) {
  const PagedCache& c = a.c;
  switch (word_bytes({(int64_t)c.channels * c.esize, address(c.k), c.k_page, c.k_slot, c.k_head,
                      address(c.v), c.v_page, c.v_slot, c.v_head, address(a.key), a.key_sb,
                      a.key_st, a.key_sh, address(a.value), a.value_sb, a.value_st, a.value_sh})) {
    case 16: return append<uint4>(a, stream);
    case 8: return append<uint2>(a, stream);
    case 4: return append<uint32_t>(a, stream);
    default: return append<uint16_t>(a, stream);
  }
}

int launch_cache_evict(const CacheEvictArgs& a, cudaStream_t stream) {
  const PagedCache& c = a.c;
  evict_select_kernel<<<(unsigned)(a.B * c.heads), EVICT_THREADS, 0, stream>>>(a);
  int st = launch_status();
  if (st != TP_OK) return st;
  switch (word_bytes({(int64_t)c.channels * c.esize, address(c.k), c.k_page, c.k_slot, c.k_head,
                      address(c.v), c.v_page, c.v_slot, c.v_head})) {
    case 16: return move<uint4>(a, stream);
    case 8: return move<uint2>(a, stream);
    case 4: return move<uint32_t>(a, stream);
    default: return move<uint16_t>(a, stream);
  }
}

}  // namespace tp
