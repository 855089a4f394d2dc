// paged_cache.cu -- what surrounds paged attention: its workspace and choice of kernels,
// writing of prompts into the pages, and eviction from them by accumulated attention weight.
#include <algorithm>

#include "cluster.cuh"
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
// A warp's lanes go along the words of (token, head) rows; one word of key and value each.  Bound
// by the bytes read and written: 8 x 1024 to 2048 tokens of 8 heads of 128 bf16 channels 20.6 us
// (4.9 TB/s).
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

// A cluster of blocks per sequence and key head: the kept slots, in order, and their mass.  Blocks
// take parts of the slots next to one another, EVICT_PER for a thread, in registers (and chunks of
// that, where the slots are more).  The place of the last kept slot among the old ones is found by
// digits of 8 bits from the top: each block counts its own, and adds up all blocks' counts (integers:
// any order of the atomics gives the same).  Then every warp's kept slots are counted by ballots, the
// counts summed in the order of the slots, and written.  What bounds it is instructions, so few rows
// go over many SMs (16 rows of 32768 slots in a block each: 31 us).
constexpr int EVICT_THREADS = 256, EVICT_PER = 16;

__global__ void __launch_bounds__(EVICT_THREADS) evict_select_kernel(const CacheEvictArgs a, int cluster) {
  constexpr int THREADS = EVICT_THREADS, WARPS = THREADS / 32, PART = THREADS * EVICT_PER;
  __shared__ int hist[2][256], merged[256];
  __shared__ u64 counts[EVICT_PER * WARPS], sums[WARPS];
  __shared__ u64 of_block[2][MAX_CLUSTER];
  __shared__ uint32_t s_digit;
  __shared__ int s_left;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster_rank();
  const int row_index = blockIdx.x / cluster, kvh = row_index % a.c.heads, b = row_index / a.c.heads;
  const int given = __ldg(a.lengths + b);
  const bool bad = given < 0 || given > a.capacity;
  if (bad && tid == 0) tp_record_index_error(a.bad.error, a.bad.seen);
  const int n = bad ? 0 : given;
  const float* row = a.mass + (int64_t)b * a.mass_sb + (int64_t)kvh * a.mass_sh;
  float* out = a.out + (int64_t)b * a.out_sb + (int64_t)kvh * a.out_sh;
  int* kept = a.kept + (int64_t)row_index * a.keep;
  if (n <= a.keep) {               // (all blocks of the cluster alike)
    for (int i = rank * THREADS + tid; i < a.keep; i += cluster * THREADS) {
      kept[i] = i < n ? i : -1;
      if (i < n && out != row) out[i] = row[i];
    }
    return;
  }
  cluster_arrive();
  // slots before `old` compete for `need` places
  const int old = n - min(a.recent, n), need = a.keep - (n - old), chunk = cluster * PART;
  float v[EVICT_PER];              // slots base + rank * PART + k * THREADS + tid
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < EVICT_PER; ++k) {
      const int64_t i = (int64_t)base + rank * PART + k * THREADS + tid;
      v[k] = i < n ? row[i] : 0.0f;
    }
  };
  // this block's slots of a chunk, in steps of THREADS
  auto steps = [&](int base, int end) {
    const int64_t some = (int64_t)end - base - (int64_t)rank * PART;
    return some <= 0 ? 0 : (int)min((int64_t)EVICT_PER, (some + THREADS - 1) / THREADS);
  };
  uint32_t prefix = 0;
  int left = need;                 // places among the slots whose high bits are `prefix`
  load(0);
  cluster_wait();                  // every block of the cluster runs
  if (need > 0) {
    hist[0][tid] = 0;
    __syncthreads();
    for (int round = 0; round < 4; ++round) {
      const int shift = 24 - 8 * round;
      int* const mine = hist[round & 1];
      for (int64_t base = 0; base < old; base += chunk) {
        if (old > chunk) load((int)base);
        const int in_use = steps((int)base, old);
#pragma unroll
        for (int k = 0; k < EVICT_PER; ++k) {
          if (k >= in_use) continue;
          const uint32_t u = ordered_bits(v[k]);
          if (base + rank * PART + k * THREADS + tid < old &&
              (round == 0 || (u >> (shift + 8)) == (prefix >> (shift + 8))))
            atomicAdd(&mine[(u >> shift) & 255], 1);
        }
      }
      cluster_sync();              // every block has counted, and read the counts before these
      hist[(round + 1) & 1][tid] = 0;
      int sum = 0;
      for (int r = 0; r < cluster; ++r) sum += (int)remote_load(remote(&mine[tid], r));
      merged[tid] = sum;
      __syncthreads();
      if (tid < 32) {              // the digit where the sum from above passes `left`
        int some[8], all = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) all += some[k] = merged[255 - (tid * 8 + k)];
        int above = all;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int y = __shfl_up_sync(0xffffffffu, above, o);
          if (tid >= o) above += y;
        }
        above -= all;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (above < left && above + some[k] >= left) {
            s_digit = (uint32_t)(255 - (tid * 8 + k));
            s_left = left - above;
          }
          above += some[k];
        }
      }
      __syncthreads();
      prefix |= s_digit << shift;
      left = s_left;
    }
  }
  // in order of the slots: those above `prefix`, the first `left` of those equal to it, and
  // the recent ones.  (A chunk is in all blocks' registers before any of it is written, and what it
  // writes is not behind it: `out` may be the mass itself.)
  int taken = 0, tied = 0, turn = 0;       // of the chunks before
  for (int64_t base = 0; base < n; base += chunk, turn ^= 1) {
    if (n > chunk) load((int)base);
    const int in_use = steps((int)base, n);
    uint32_t sure = 0, tie = 0;            // of this thread's slots, a bit each
#pragma unroll
    for (int k = 0; k < EVICT_PER; ++k) {
      u64 both = 0;
      if (k < in_use) {
        const int64_t i = base + rank * PART + k * THREADS + tid;
        const uint32_t u = ordered_bits(v[k]);
        const bool s = i < n && (i >= old || (need > 0 && u > prefix));
        const bool t = i < old && need > 0 && u == prefix;
        sure |= (uint32_t)s << k;
        tie |= (uint32_t)t << k;
        both = (u64)__popc(__ballot_sync(0xffffffffu, s)) << 32 | __popc(__ballot_sync(0xffffffffu, t));
      }
      if (lane == 0) counts[k * WARPS + warp] = both;
    }
    __syncthreads();
    // the warps' counts of all steps, summed over those before
    u64 upto = tid < EVICT_PER * WARPS ? counts[tid] : 0;
    const u64 one = upto;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    u64 before = 0, mine = 0;
    for (int w = 0; w < WARPS; ++w) {
      before += w < warp ? sums[w] : 0;
      mine += sums[w];
    }
    if (tid < cluster) remote_store(remote(&of_block[turn][rank], tid), mine);
    cluster_sync();                        // (a chunk on, the other half is written: read by then)
    u64 earlier = 0, whole = 0;
    for (int r = 0; r < cluster; ++r) {
      earlier += r < rank ? of_block[turn][r] : 0;
      whole += of_block[turn][r];
    }
    if (tid < EVICT_PER * WARPS) counts[tid] = earlier + before + upto - one;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EVICT_PER; ++k) {
      if (k >= in_use) continue;
      const u64 first = counts[k * WARPS + warp];
      const bool t = tie >> k & 1;
      const unsigned ties = __ballot_sync(0xffffffffu, t), low = (1u << lane) - 1;
      const int tie_rank = tied + (int)(uint32_t)first + __popc(ties & low);
      const unsigned sures = __ballot_sync(0xffffffffu, sure >> k & 1);
      const int place = taken + (int)(first >> 32) + __popc(sures & low) + min(tie_rank, left);
      if ((sure >> k & 1) || (t && tie_rank < left)) {
        kept[place] = (int)base + rank * PART + k * THREADS + tid;
        out[place] = v[k];
      }
    }
    taken += (int)(whole >> 32);
    tied += (int)(uint32_t)whole;
    __syncthreads();
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
// LOOK: rows of a batch that a thread looks up.
template <typename W, int LOOK>
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
  const int batch = per * MOVE_DEPTH;          // rows; at most LOOK * MOVE_THREADS
  const int batches = (a.keep + batch - 1) / batch;

  int slot[LOOK], after[LOOK], from_page[LOOK], to_page[LOOK];
  auto ask_slots = [&](int t, int (&into)[LOOK]) {
#pragma unroll
    for (int k = 0; k < LOOK; ++k) {
      const int in = threadIdx.x + k * MOVE_THREADS, i = t * batch + in;
      into[k] = in < batch && t < batches && i < a.keep ? kept[i] : -1;
    }
  };
  auto ask_pages = [&](int t) {                // of batch t, whose slots are in `slot`
#pragma unroll
    for (int k = 0; k < LOOK; ++k) {
      const int i = t * batch + threadIdx.x + k * MOVE_THREADS;
      if (slot[k] < 0 || slot[k] == i) continue;
      from_page[k] = __ldg(row + a.c.column(slot[k]));
      to_page[k] = __ldg(row + a.c.column(i));
    }
  };
  auto note = [&](int t) {                     // batch t's rows into the ring; on to the next slots
    RowMove* const to = ring + t % 3 * batch;
#pragma unroll
    for (int k = 0; k < LOOK; ++k) {
      const int in = threadIdx.x + k * MOVE_THREADS, i = t * batch + in;
      if (in < batch) {
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
      slot[k] = after[k];
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
  ask_slots(0, slot);
  for (int t = 0; t < 2; ++t) {
    ask_slots(t + 1, after);
    ask_pages(t);
    note(t);
  }
  __syncthreads();
  read(0, x);
  for (int t = 0; t < batches; ++t) {
    ask_slots(t + 3, after);
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
    __syncthreads();
  }
}

template <typename W>
int move(const CacheEvictArgs& a, cudaStream_t stream) {
  // a row of words for the lanes next to one another, down to 64 bytes of it where sequences and
  // heads are few (32 x 8 heads of 128-byte rows: 27.8 us by whole rows, 33.2 by halves)
  const int words = a.c.channels * a.c.esize / (int)sizeof(W), least = std::max(1, 64 / (int)sizeof(W));
  int width = std::min(words, MOVE_THREADS / 4);
  while (width > least && a.B * a.c.heads * 2 * ceil_div(words, width) < 2 * num_sms()) width = (width + 1) / 2;
  const int slices = (words + width - 1) / width;
  const int64_t blocks = a.B * a.c.heads * 2 * slices;
  TP_RETURN_IF(blocks > INT32_MAX, TP_ERR_TOO_LARGE);
  const size_t smem = (size_t)3 * (MOVE_THREADS / width) * MOVE_DEPTH * sizeof(RowMove);
  constexpr int FEW = 2;                 // (8 rows a thread looked up leave the others no registers)
  auto* kernel = width * FEW >= MOVE_DEPTH ? evict_move_kernel<W, FEW> : evict_move_kernel<W, MOVE_DEPTH>;
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
  // (16 rows of 32768 slots: both kernels 51 us with clusters of eight, over 100 with single blocks)
  int cluster = 1;
  while (cluster < MAX_CLUSTER && a.capacity > cluster * EVICT_THREADS * EVICT_PER &&
         a.B * c.heads * cluster * 2 <= 8 * num_sms())
    cluster *= 2;
  const int st = launch_clusters(evict_select_kernel, a.B * c.heads * cluster, EVICT_THREADS, cluster,
                                 stream, a, cluster);
  if (st != TP_OK || c.channels == 0) return st;       // (rows without a channel: none to move)
  switch (word_bytes({(int64_t)c.channels * c.esize, address(c.k), c.k_page, c.k_slot, c.k_head,
                      address(c.v), c.v_page, c.v_slot, c.v_head})) {
    case 16: return move<uint4>(a, stream);
    case 8: return move<uint2>(a, stream);
    case 4: return move<uint32_t>(a, stream);
    default: return move<uint16_t>(a, stream);
  }
}

}  // namespace tp
