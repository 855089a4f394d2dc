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

// One block per sequence and key head: the kept slots, in order, and their mass.  The mass is read
// once where it fits shared memory (STAGED slots).  The place of the last kept slot among the old
// ones is found by digits of 11, 11 and 10 bits from the top (integer counts: any order of the
// atomics gives the same; of 8 bits, nearly all slots would meet in a few counters); then each
// warp counts what it keeps of its part, and writes it.
constexpr int STAGED = 49152, DIGITS = 2048;

template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const CacheEvictArgs a, int staged) {
  constexpr int WARPS = THREADS / 32, EACH = DIGITS / THREADS;
  extern __shared__ float stage[];
  __shared__ int hist[DIGITS];
  __shared__ int sums[2][WARPS];
  __shared__ uint32_t s_digit;
  __shared__ int s_left;
  const int kvh = blockIdx.x % a.c.heads, b = blockIdx.x / a.c.heads, tid = threadIdx.x, lane = tid & 31,
            warp = tid >> 5;
  const int given = __ldg(a.lengths + b);
  const bool bad = given < 0 || given > a.capacity;
  if (bad && tid == 0) tp_record_index_error(a.bad.error, a.bad.seen);
  const int n = bad ? 0 : given;
  const float* row = a.mass + (int64_t)b * a.mass_sb + (int64_t)kvh * a.mass_sh;
  float* out = a.out + (int64_t)b * a.out_sb + (int64_t)kvh * a.out_sh;
  int* kept = a.kept + (int64_t)blockIdx.x * a.keep;
  if (n <= a.keep) {
    for (int i = tid; i < a.keep; i += THREADS) {
      kept[i] = i < n ? i : -1;
      if (i < n && out != row) out[i] = row[i];
    }
    return;
  }
  const bool in_smem = n <= staged;
  if (in_smem)
    for (int i = tid; i < n; i += THREADS) stage[i] = row[i];
  const float* mass = in_smem ? stage : row;
  // slots before `old` compete for `need` places
  const int old = n - min(a.recent, n), need = a.keep - (n - old);
  uint32_t prefix = 0;
  int left = need;                 // places among the slots whose high bits are `prefix`
  if (need > 0) {
    for (int round = 0; round < 3; ++round) {
      const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
      for (int i = tid; i < DIGITS; i += THREADS) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < old; i += THREADS) {
        const uint32_t u = ordered_bits(mass[i]);
        if (round == 0 || (u >> (shift + bits)) == (prefix >> (shift + bits)))
          atomicAdd(&hist[(u >> shift) & ((1u << bits) - 1)], 1);
      }
      __syncthreads();
      // the digit where the sum from above passes `left`
      int mine[EACH], all = 0;
#pragma unroll
      for (int k = 0; k < EACH; ++k) all += mine[k] = hist[DIGITS - 1 - (tid * EACH + k)];
      int above = all;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += y;
      }
      if (lane == 31) sums[0][warp] = above;
      __syncthreads();
      above -= all;
      for (int w = 0; w < warp; ++w) above += sums[0][w];
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        if (above < left && above + mine[k] >= left) {
          s_digit = (uint32_t)(DIGITS - 1 - (tid * EACH + k));
          s_left = left - above;
        }
        above += mine[k];
      }
      __syncthreads();
      prefix |= s_digit << shift;
      left = s_left;
    }
  }
  // in order of the slots: those above `prefix`, the first `left` of those equal to it, and
  // the recent ones
  __syncthreads();                 // (mass of all slots is read before `out` is written)
  const int part = ((n + WARPS - 1) / WARPS + 31) / 32 * 32, from = min(n, warp * part), to = min(n, from + part);
  auto more = [&](uint32_t u, int i) { return i >= old || (need > 0 && u > prefix); };
  auto equal = [&](uint32_t u, int i) { return i < old && need > 0 && u == prefix; };
  int sure = 0, ties = 0;
  for (int base = from; base < to; base += 32) {
    const int i = base + lane;
    const uint32_t u = i < to ? ordered_bits(mass[i]) : 0;
    sure += __popc(__ballot_sync(0xffffffffu, i < to && more(u, i)));
    ties += __popc(__ballot_sync(0xffffffffu, i < to && equal(u, i)));
  }
  if (lane == 0) {
    sums[0][warp] = sure;
    sums[1][warp] = ties;
  }
  __syncthreads();
  int at = 0, tie = 0;
  for (int w = 0; w < warp; ++w) {
    at += sums[0][w];
    tie += sums[1][w];
  }
  at += min(tie, left);
  // A warp's part may be written while another's is still to be read: only where mass is staged,
  // or `out` is another tensor, may all go on at once.
  const bool apart = in_smem || out != row;
  for (int turn = 0; turn < (apart ? 1 : WARPS); ++turn) {
    if (!apart) __syncthreads();
    if (apart || turn == warp)
      for (int base = from; base < to; base += 32) {
        const int i = base + lane;
        const float m = i < to ? mass[i] : 0.0f;
        const uint32_t u = ordered_bits(m);
        const unsigned is_tie = __ballot_sync(0xffffffffu, i < to && equal(u, i));
        const bool mine = i < to && equal(u, i) && tie + __popc(is_tie & ((1u << lane) - 1)) < left;
        const bool take = i < to && (more(u, i) || mine);
        const unsigned takers = __ballot_sync(0xffffffffu, take);
        const int place = at + __popc(takers & ((1u << lane) - 1));
        if (take) {
          kept[place] = i;
          out[place] = m;
        }
        at += __popc(takers);
        tie += __popc(is_tie);
      }
  }
}

// Moves kept rows to the front.  Different words of a row move apart from one another: a block
// takes some words of all kept rows of a sequence and head, in order.  Row i comes from kept[i] >= i,
// so a batch's rows are read before any of them is written (one barrier), and no later batch reads
// what an earlier one wrote.  While a batch is written, the rows of the next one are under way, the
// pages of the one after it and the slots of the third: one latency per batch instead of three
// (2 x 8 heads of 8192 rows of 128 bf16 channels, slots, pages and rows in turn: 59 us).
constexpr int MOVE_THREADS = 512, MOVE_DEPTH = 8;
struct RowMove {
  int64_t from, to;                // in bytes from the head's first row; -1: stays
};
template <typename W>
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const CacheEvictArgs a, int words,
                                                                  int width, int slices) {
  extern __shared__ __align__(16) RowMove ring[];      // three batches
  asm volatile("griddepcontrol.wait;" ::: "memory");
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
  const int w = slice * width + threadIdx.x % width;
  char* const base = (value ? a.c.v + kvh * a.c.v_head : a.c.k + kvh * a.c.k_head) + w * (int)sizeof(W);
  const int64_t page_bytes = value ? a.c.v_page : a.c.k_page, slot_bytes = value ? a.c.v_slot : a.c.k_slot;
  const int per = MOVE_THREADS / width, mine = threadIdx.x / width;
  const bool active = mine < per && w < words;
  const int batch = per * MOVE_DEPTH;          // rows; at most MOVE_DEPTH for a thread to look up
  const int batches = (a.keep + batch - 1) / batch;

  int slot[MOVE_DEPTH], from_page[MOVE_DEPTH], to_page[MOVE_DEPTH];
  auto ask_slots = [&](int t) {
#pragma unroll
    for (int k = 0; k < MOVE_DEPTH; ++k) {
      const int in = threadIdx.x + k * MOVE_THREADS, i = t * batch + in;
      slot[k] = in < batch && i < a.keep && t < batches ? kept[i] : -1;
    }
  };
  auto ask_pages = [&](int t) {
#pragma unroll
    for (int k = 0; k < MOVE_DEPTH; ++k) {
      const int i = t * batch + threadIdx.x + k * MOVE_THREADS;
      if (slot[k] < 0 || slot[k] == i) continue;
      from_page[k] = __ldg(row + a.c.column(slot[k]));
      to_page[k] = __ldg(row + a.c.column(i));
    }
  };
  auto note = [&](int t) {                     // batch t's rows into the ring
    RowMove* const to = ring + t % 3 * batch;
#pragma unroll
    for (int k = 0; k < MOVE_DEPTH; ++k) {
      const int in = threadIdx.x + k * MOVE_THREADS, i = t * batch + in;
      if (in >= batch) continue;
      RowMove m{-1, -1};
      if (slot[k] >= 0 && slot[k] != i) {
        if (from_page[k] < 0 || from_page[k] >= a.c.pages || to_page[k] < 0 || to_page[k] >= a.c.pages) {
          tp_record_index_error(a.bad.error, a.bad.seen);
        } else {
          m.from = from_page[k] * page_bytes + a.c.within(slot[k], a.c.column(slot[k])) * slot_bytes;
          m.to = to_page[k] * page_bytes + a.c.within(i, a.c.column(i)) * slot_bytes;
        }
      }
      to[in] = m;
    }
  };
  W x[MOVE_DEPTH], y[MOVE_DEPTH];
  auto read = [&](int t, W (&into)[MOVE_DEPTH]) {
    if (!active || t >= batches) return;
#pragma unroll
    for (int k = 0; k < MOVE_DEPTH; ++k) {
      const int64_t from = ring[t % 3 * batch + k * per + mine].from;
      if (from >= 0) into[k] = *(const W*)(base + from);
    }
  };
  for (int t = 0; t < 2; ++t) {
    ask_slots(t);
    ask_pages(t);
    note(t);
  }
  ask_slots(2);
  __syncthreads();
  read(0, x);
  for (int t = 0; t < batches; ++t) {
    ask_pages(t + 2);
    read(t + 1, y);
    __syncthreads();                           // batch t has been read by all
    if (active)
#pragma unroll
      for (int k = 0; k < MOVE_DEPTH; ++k) {
        const int64_t to = ring[t % 3 * batch + k * per + mine].to;
        if (to >= 0) *(W*)(base + to) = x[k];
        x[k] = y[k];
      }
    note(t + 2);
    ask_slots(t + 3);
    __syncthreads();
  }
}

template <typename W>
int move(const CacheEvictArgs& a, cudaStream_t stream) {
  // a row of words for the lanes next to one another, down to 64 bytes of it where sequences and
  // heads are few
  const int words = a.c.channels * a.c.esize / (int)sizeof(W), least = std::max(1, 64 / (int)sizeof(W));
  int width = std::min(words, MOVE_THREADS / 4);
  while (width > least && a.B * a.c.heads * 2 * ceil_div(words, width) < 2 * num_sms()) width = (width + 1) / 2;
  const int slices = (words + width - 1) / width;
  const int64_t blocks = a.B * a.c.heads * 2 * slices;
  TP_RETURN_IF(blocks > INT32_MAX, TP_ERR_TOO_LARGE);
  const size_t smem = (size_t)3 * (MOVE_THREADS / width) * MOVE_DEPTH * sizeof(RowMove);
  auto* kernel = evict_move_kernel<W>;
  const int st = allow_smem((const void*)kernel, smem);
  if (st != TP_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(MOVE_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, a, words, width, slices));
}

template <int THREADS>
int select(const CacheEvictArgs& a, cudaStream_t stream) {
  const int staged = std::min(a.capacity, STAGED);
  auto* kernel = evict_select_kernel<THREADS>;
  const int st = allow_smem((const void*)kernel, (size_t)staged * 4);
  if (st != TP_OK) return st;
  kernel<<<(unsigned)(a.B * a.c.heads), THREADS, (size_t)staged * 4, stream>>>(a, staged);
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
  const int st = a.capacity <= 4096 ? select<256>(a, stream) : select<1024>(a, stream);
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
