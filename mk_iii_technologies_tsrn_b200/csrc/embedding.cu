// embedding.cu -- the token embedding of a language model and its gradient:
//
//   out[i] = weight[id_i] * scale (+ pos_weight[position_i])
//   dweight[v] = scale * sum over i with id_i = v of dout[i]
//
// as `embed(ids) * sqrt(d_model) + pos_embed(positions)` of the token models
// (tropformer_dropin.py:616-720).  An id or position outside its table is
// never read: the token's row of `out` is NaN, its row of dout adds to neither
// table's gradient, and TP_DEVERR_INDEX is recorded in the device error word.
//
// The forward is a row gather: bound by the rows read and written.
//
// The gradient sums rows by token.  Adding them with atomics would make the
// order, and so the bits, depend on timing, and a frequent token would
// serialise; instead the tokens are sorted by id (a stable counting sort, so
// equal ids keep their order) and the sorted rows summed in that order:
//
// 1. sort: the id is cut into one or two digits (three above 2^20 rows).  Per
//    digit the tokens are counted by warp, and placed: each warp ranks its run of
//    tokens 32 at a time by digit match, on top of the counts of earlier bins,
//    blocks and warps.  Up to 2^18 tokens one cluster of up to 16 blocks does all
//    of it in one launch (65536 tokens of 256 rows 13 us, 131072 of 131072 rows
//    34 us); more take two kernels a digit over all SMs.
// 2. sum: tokens and table rows form one list of N + V items (the tokens of a
//    row, then the row's end), tokens with twice the weight.  Each team of threads
//    takes an equal share of it, found by bisection, whatever the ids: it adds a
//    row of dout per token and writes a row of the gradient (zeros for an
//    absent id) per end.  So every dout row is read once and every gradient
//    row written once: the bytes the result needs.
// 3. join: a table row whose tokens reach over several shares left fp32
//    partial sums in the workspace; they are added in order.
//
// Measured: the forward of 32 x 4096 tokens of 1024 bf16 channels 59 us, its gradient
// for 131072 rows 146 us (sum 111), together 133 us of bytes at the card's copy rate (of
// ids that fall off as 1 / rank 32600 rows are met); 64 x 1024 tokens of 640 fp32
// channels with 256 rows 33 and 65 us, 52 us of bytes.  There the sort (13 us) is a
// chain of exchanges over 16 blocks, the sum runs at half of the DRAM's rate with 19
// warps on an SM, and the join waits for its partial rows.
#include <initializer_list>

#include "maxplus_internal.cuh"
#include "rowvec.cuh"

namespace tp {

namespace {

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  return is64 ? __ldg((const long long*)p + i) : (int64_t)__ldg((const int*)p + i);
}

// ---------------------------------------------------------------- forward
// A team of `lanes` threads takes TOK tokens and UV vectors of each at a time, so
// that their loads are under way together.
template <typename T, int VEC, int TOK, int UV>
__global__ void __launch_bounds__(128) embedding_fwd_kernel(const EmbeddingArgs a, int lanes,
                                                            const IndexErrorWords bad) {
  using V = RowVec<T, VEC>;
  const int t = threadIdx.x % lanes, per = blockDim.x / lanes;
  const int64_t nv = a.D / VEC;
  for (int64_t i0 = ((int64_t)blockIdx.x * per + threadIdx.x / lanes) * TOK; i0 < a.N;
       i0 += (int64_t)gridDim.x * per * TOK) {
    const T* wr[TOK];
    const T* pr[TOK];
    bool ok[TOK];
#pragma unroll
    for (int k = 0; k < TOK; ++k) {
      const int64_t i = i0 + k < a.N ? i0 + k : i0;
      const int64_t id = load_index(a.ids, a.ids64, i);
      int64_t at = 0;
      ok[k] = id >= 0 && id < a.V;
      if (a.pos_weight) {
        at = a.positions ? load_index(a.positions, a.ids64, i) : i % a.T;
        ok[k] = ok[k] && at >= 0 && at < a.L;
      }
      if (!ok[k] && t == 0) tp_record_index_error(bad.error, bad.seen);
      wr[k] = (const T*)a.weight + (ok[k] ? id * a.ldw : 0);    // read only if ok
      pr[k] = (const T*)a.pos_weight + (ok[k] ? at * a.ldp : 0);
    }
    for (int64_t v0 = t; v0 < nv; v0 += UV * lanes) {
      V w[TOK][UV], p[TOK][UV];
#pragma unroll
      for (int k = 0; k < TOK; ++k)
#pragma unroll
        for (int u = 0; u < UV; ++u) {
          const int64_t v = v0 + u * lanes;
          w[k][u].zero();
          p[k][u].zero();
          if (ok[k] && v < nv) {
            w[k][u].load(wr[k] + v * VEC);
            if (a.pos_weight) p[k][u].load(pr[k] + v * VEC);
          }
        }
#pragma unroll
      for (int k = 0; k < TOK; ++k) {
        if (i0 + k >= a.N) break;
#pragma unroll
        for (int u = 0; u < UV; ++u) {
          const int64_t v = v0 + u * lanes;
          if (v >= nv) break;
          float f[VEC];
          w[k][u].get(f);
          if (a.pos_weight) {
            float q[VEC];
            p[k][u].get(q);
            // product and sum rounded one by one, as the unfused expression
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = __fadd_rn(__fmul_rn(f[j], a.scale), q[j]);
          } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = __fmul_rn(f[j], a.scale);
          }
          if (!ok[k]) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = __int_as_float(0x7fc00000);
          }
          V r;
          r.set(f);
          r.store((T*)a.out + (i0 + k) * a.D + v * VEC);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- sort
constexpr int SORT_THREADS = 256;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_MAX_BITS = 11;
constexpr int64_t SORT_MAX_TILES = 128;

// Lanes of the warp whose token has this lane's digit (0 where `in` is false), by
// one vote per bit: several times faster than __match_any_sync on many different
// digits.
__device__ __forceinline__ unsigned same_digit(bool in, int d, int bits) {
  unsigned m = __ballot_sync(0xffffffffu, in);
  for (int b = 0; b < bits; ++b) {
    const unsigned set = __ballot_sync(0xffffffffu, (d >> b) & 1);
    m &= (d >> b) & 1 ? set : ~set;
  }
  return in ? m : 0u;
}

struct SortPlan {
  // blocks of sort_cluster_kernel; 0: the two-kernel sort, of more than 2^18 tokens or for
  // a table of 2^30 rows
  int cluster;
  int64_t tile;     // tokens per block, a multiple of 32 * SORT_WARPS
  int tiles;
  int passes, bits; // digits per key, bits per digit
};

SortPlan sort_plan(int64_t N, int64_t V) {
  SortPlan p;
  int bits = 1;
  while (((int64_t)1 << bits) <= V) ++bits;     // keys 0 .. V (V: not in the table)
  p.cluster = 0;
  const int most = N <= ((int64_t)1 << 18) ? 10 : SORT_MAX_BITS;
  p.passes = (bits + most - 1) / most;
  if (most == 10 && p.passes <= 3) {
    p.cluster = 1;         // a block per 4096 tokens
    while (p.cluster < 16 && (int64_t)p.cluster * 4096 < N) p.cluster *= 2;
  } else {
    p.passes = (bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
  }
  p.bits = (bits + p.passes - 1) / p.passes;
  const int64_t unit = 32 * SORT_WARPS;
  p.tile = N > 0 ? ceil_div(ceil_div(N, SORT_MAX_TILES), unit) * unit : unit;
  p.tiles = (int)ceil_div(N, p.tile);
  return p;
}

// A token's index in this table, and in the other one where it has one.
struct Keys {
  const void* ids;
  const void* other;      // NULL: no other table
  int ids64;              // of both
  int64_t V, padding_idx, other_rows;
};

struct SortArgs {
  Keys keys;              // first pass
  const int2* in;         // later passes: (key, token) of the pass before
  int2* out;
  int* hist;              // [tiles][bins]
  int64_t N, tile;
  int tiles, shift, bins, bits;
  int first;
};

// V for a token that is not in both tables or gets no gradient: sorted behind the rows
__device__ __forceinline__ int key_of(const Keys& k, int64_t i) {
  const int64_t id = load_index(k.ids, k.ids64, i);
  bool in = id >= 0 && id < k.V && id != k.padding_idx;
  if (k.other != nullptr) {
    const int64_t o = load_index(k.other, k.ids64, i);
    in = in && o >= 0 && o < k.other_rows;
  }
  return in ? (int)id : (int)k.V;
}

__device__ __forceinline__ int sort_key(const SortArgs& s, int64_t i) {
  return s.first ? key_of(s.keys, i) : s.in[i].x;
}

__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const SortArgs s) {
  extern __shared__ int s_cnt[];
  for (int b = threadIdx.x; b < s.bins; b += SORT_THREADS) s_cnt[b] = 0;
  __syncthreads();
  const int64_t lo = blockIdx.x * s.tile, hi = min(s.N, lo + s.tile);
  for (int64_t i = lo + threadIdx.x; i < hi; i += SORT_THREADS)
    atomicAdd(&s_cnt[(sort_key(s, i) >> s.shift) & (s.bins - 1)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < s.bins; b += SORT_THREADS)
    s.hist[(int64_t)blockIdx.x * s.bins + b] = s_cnt[b];
}

// Exclusive sum over the block's threads; total in *total.
__device__ __forceinline__ int block_exclusive(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SORT_WARPS; ++w) {
    if (w < warp) before += s_warp[w];
    all += s_warp[w];
  }
  *total = all;
  return before + inc - v;
}

__global__ void __launch_bounds__(SORT_THREADS) sort_place_kernel(const SortArgs s) {
  extern __shared__ int s_mem[];     // [SORT_WARPS][bins]: next place of each warp and bin
  __shared__ int s_warp[SORT_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* mine = s_mem + warp * s.bins;
  for (int b = threadIdx.x; b < SORT_WARPS * s.bins; b += SORT_THREADS) s_mem[b] = 0;
  __syncthreads();
  // counts of this tile by warp
  const int64_t run = s.tile / SORT_WARPS;
  const int64_t lo = blockIdx.x * s.tile + warp * run, hi = min(s.N, lo + run);
  for (int64_t i = lo + lane; i < hi; i += 32)
    atomicAdd(&mine[(sort_key(s, i) >> s.shift) & (s.bins - 1)], 1);
  __syncthreads();
  // start of each bin: all tokens of lower bins, then this bin's of earlier tiles
  int base = 0;
  for (int b0 = 0; b0 < s.bins; b0 += SORT_THREADS) {
    const int b = b0 + threadIdx.x;
    int all = 0, earlier = 0;
    if (b < s.bins) {
#pragma unroll 8
      for (int t = 0; t < s.tiles; ++t) {
        const int n = s.hist[(int64_t)t * s.bins + b];
        all += n;
        if (t < (int)blockIdx.x) earlier += n;
      }
    }
    int total;
    int at = base + block_exclusive(all, s_warp, &total) + earlier;
    base += total;
    if (b < s.bins) {
#pragma unroll
      for (int w = 0; w < SORT_WARPS; ++w) {
        const int n = s_mem[w * s.bins + b];
        s_mem[w * s.bins + b] = at;
        at += n;
      }
    }
  }
  __syncthreads();
  // place this warp's run in order, 32 tokens at a time
  for (int64_t i0 = lo; i0 < hi; i0 += 32) {
    const int64_t i = i0 + lane;
    const bool in = i < hi;
    const int key = in ? sort_key(s, i) : -1;
    const int d = in ? (key >> s.shift) & (s.bins - 1) : 0;
    const unsigned same = same_digit(in, d, s.bits);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int at = 0;
    if (in) at = mine[d] + rank;
    __syncwarp();
    if (in) {
      if (rank == 0) mine[d] += __popc(same);
      s.out[at] = make_int2(key, s.first ? (int)i : s.in[i].y);
    }
    __syncwarp();
  }
}

// The whole sort in one launch: a cluster of S blocks of 32 warps, each warp a
// contiguous run of tokens.  The blocks exchange their counts and their output
// through global memory (L2), with a cluster barrier between.
constexpr int SC_THREADS = 1024, SC_WARPS = 32;
constexpr int SC_MAX_BITS = 10;
constexpr int SC_GROUPS = 4;

struct ClusterSortArgs {
  Keys keys;
  int2* pairs[2];         // (key, token)
  int* hist;              // [passes][S][bins]
  int64_t N;
  int passes, bits, S;
};

__device__ __forceinline__ void sc_cluster_sync(int S) {
  if (S > 1)
    asm volatile(
        "barrier.cluster.arrive.release.aligned;\n\t"
        "barrier.cluster.wait.acquire.aligned;" ::
            : "memory");
  else
    __syncthreads();
}

__global__ void __launch_bounds__(SC_THREADS) sort_cluster_kernel(const ClusterSortArgs s) {
  extern __shared__ uint16_t s_runs[];          // [SC_WARPS][bins]: of a warp, then before it
  __shared__ int s_base[1 << SC_MAX_BITS], s_warp[SC_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int bins = 1 << s.bits;
  const int64_t share = ceil_div(s.N, (int64_t)s.S);
  const int64_t run = ceil_div(share, (int64_t)(32 * SC_WARPS)) * 32;   // tokens of a warp
  const int64_t lo = min(s.N, ((int64_t)blockIdx.x * SC_WARPS + warp) * run);
  const int64_t hi = min(s.N, lo + run);
  uint16_t* const mine = s_runs + warp * bins;
  for (int pass = 0; pass < s.passes; ++pass) {
    const int2* const in_pairs = s.pairs[(pass & 1) ^ 1];
    int2* const out_pairs = s.pairs[pass & 1];
    const int shift = pass * s.bits;
    auto pair_at = [&](int64_t i) {
      if (pass > 0) return __ldcg(in_pairs + i);
      return make_int2(key_of(s.keys, i), (int)i);
    };
    for (int b = threadIdx.x; b < SC_WARPS * bins / 2; b += SC_THREADS)
      reinterpret_cast<unsigned*>(s_runs)[b] = 0;
    __syncthreads();
    // counts of this warp's run (16 bits each, two in a word)
    for (int64_t i0 = lo; i0 < hi; i0 += 32 * SC_GROUPS) {
      int key[SC_GROUPS];
#pragma unroll
      for (int k = 0; k < SC_GROUPS; ++k)
        key[k] = i0 + k * 32 + lane < hi ? pair_at(i0 + k * 32 + lane).x : -1;
#pragma unroll
      for (int k = 0; k < SC_GROUPS; ++k) {
        const int d = (key[k] >> shift) & (bins - 1);
        if (key[k] >= 0)
          atomicAdd(reinterpret_cast<unsigned*>(mine) + (d >> 1), 1u << ((d & 1) * 16));
      }
    }
    __syncthreads();
    int* const hist = s.hist + (int64_t)pass * s.S * bins;
    for (int b = threadIdx.x; b < bins; b += SC_THREADS) {
      int n = 0;
#pragma unroll 8
      for (int w = 0; w < SC_WARPS; ++w) {
        const int c = s_runs[w * bins + b];
        s_runs[w * bins + b] = (uint16_t)n;     // at most 2^18 / 16 tokens in a block
        n += c;
      }
      __stcg(hist + blockIdx.x * bins + b, n);
    }
    sc_cluster_sync(s.S);
    // start of each bin: all tokens of lower bins, then this bin's of earlier blocks
    // (at most as many bins as threads)
    int all = 0, earlier = 0;
    if (threadIdx.x < bins) {
#pragma unroll 4
      for (int q = 0; q < s.S; ++q) {
        const int n = __ldcg(hist + q * bins + threadIdx.x);
        all += n;
        if (q < (int)blockIdx.x) earlier += n;
      }
    }
    int inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      int v = s_warp[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      s_warp[lane] = v;
    }
    __syncthreads();
    if (threadIdx.x < bins)
      s_base[threadIdx.x] = (warp > 0 ? s_warp[warp - 1] : 0) + inc - all + earlier;
    __syncthreads();
    // place this warp's run in order
    for (int64_t i0 = lo; i0 < hi; i0 += 32 * SC_GROUPS) {
      int2 pair[SC_GROUPS];
#pragma unroll
      for (int k = 0; k < SC_GROUPS; ++k) {
        const int64_t i = i0 + k * 32 + lane;
        pair[k] = i < hi ? pair_at(i) : make_int2(-1, 0);
      }
#pragma unroll
      for (int k = 0; k < SC_GROUPS; ++k) {
        if (i0 + k * 32 >= hi) break;
        const bool in = pair[k].x >= 0;
        const int d = in ? (pair[k].x >> shift) & (bins - 1) : 0;
        const unsigned same = same_digit(in, d, s.bits);
        const int rank = __popc(same & ((1u << lane) - 1u));
        int at = 0;
        if (in) at = s_base[d] + mine[d] + rank;
        __syncwarp();
        if (in) {
          if (rank == 0) mine[d] += (uint16_t)__popc(same);
          __stcg(out_pairs + at, pair[k]);
        }
        __syncwarp();
      }
    }
    if (pass + 1 < s.passes) sc_cluster_sync(s.S);
  }
}

// Up to 1024 tokens: one block, each thread counts the tokens before its own.
constexpr int64_t SMALL_TOKENS = 1024;
__global__ void __launch_bounds__(SMALL_TOKENS) sort_small_kernel(const Keys keys, int N,
                                                                  int2* out) {
  __shared__ __align__(16) int s_key[SMALL_TOKENS];
  const int i = threadIdx.x;
  const int key = i < N ? key_of(keys, i) : 0x7fffffff;
  s_key[i] = key;
  __syncthreads();
  if (i >= N) return;
  int rank = 0;
  for (int j = 0; j < N; j += 4) {        // (places behind N hold the largest key)
    const int4 k = *reinterpret_cast<const int4*>(s_key + j);
    rank += (k.x < key || (k.x == key && j < i)) + (k.y < key || (k.y == key && j + 1 < i)) +
            (k.z < key || (k.z == key && j + 2 < i)) + (k.w < key || (k.w == key && j + 3 < i));
  }
  out[rank] = make_int2(key, i);
}

// ---------------------------------------------------------------- sum
struct SumArgs {
  const int2* pairs;    // (key, token), sorted by key; V: dropped
  int64_t N, V, D;
  const void* dout;
  float scale;
  void* dweight;
  int64_t share;        // items per team
  int64_t shares;
  int lanes;            // threads of a team
  float* head;          // [shares][D]: end of a row begun in an earlier share
  float* tail;          // [shares][D]: begin of a row that ends in a later share
  int64_t* rows;        // [shares]: the first row of the share
  int* flags;           // [shares]: bit 0 the first row began earlier, bit 1 an end lies inside
};

// The list of the tokens of row 0, the end of row 0, the tokens of row 1, ..., a token
// TOKEN_COST places long and a row end one: token j begins at keys[j] + cost * j.  A
// token is a row read, mostly one latency after the other within a team, an end a row
// written: where frequent ids leave some teams with tokens alone and others with absent
// rows, shares of equal counts wait for the former (8604 tokens of 132453 rows of 1096
// fp32 channels, Zipf's law: 181 us at 1, 136 us at 2; 32 x 4096 of 131072 rows of 1024
// bf16 channels: 126 and 111 us).
constexpr int64_t TOKEN_COST = 2;
// Tokens that begin before place `d`: the smallest j with keys[j] + cost * j >= d.  A
// whole warp searches, 32 places at a time.
__device__ __forceinline__ int64_t tokens_before(const int2* pairs, int64_t N, int64_t d) {
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, hi = min(N, d);            // the answer lies in [lo, hi]
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32;
    const int64_t at = lo + lane * step;     // 32 places cover [lo, hi)
    const bool below = at < hi && (int64_t)__ldg(pairs + at).x + TOKEN_COST * at < d;
    const int n = __popc(__ballot_sync(0xffffffffu, below));   // below for the first n lanes
    if (n == 0) return lo;
    const int64_t last = lo + (n - 1) * step;                  // the last place known below
    hi = min(hi, last + step);
    lo = last + 1;
  }
  return lo;
}

// fp32 rows come through shared memory: SUM_STAGES batches of SUM_BATCH under way, a
// thread's 16 bytes of each in a place of its own (64 x 1024 tokens of 256 rows of 640
// channels, the gradient with its sort: 67 us, against 82 us with eight rows at a time
// in registers, 70 with three batches and more threads, 73 with six and fewer).  bf16
// rows have half the bytes for the same steps and take eight at a time in registers
// (the same tokens: 56 us against 71; 60 x 4096 of 32000 rows of 768: 149 against 195).
constexpr int SUM_BATCH = 4, SUM_STAGES = 4;
template <typename T, int VEC>
constexpr bool SUM_ASYNC = VEC * sizeof(T) == 16 && sizeof(T) == 4;
constexpr int SUM_CHUNK = 128;     // pairs at a time, of rows loaded to registers

// Zeros to elements [lo, hi) of out with `lanes` threads: whole 16 bytes wherever the
// range holds them, since rows of absent tokens lie one behind the other.
template <typename T>
__device__ __forceinline__ void fill_zeros(T* out, int64_t lo, int64_t hi, int t, int lanes) {
  constexpr int W = 16 / sizeof(T);
  T* p = out + lo;
  int64_t n = hi - lo;
  const int64_t head =
      min(n, (int64_t)((16 - ((uintptr_t)p & 15)) & 15) / (int64_t)sizeof(T));
  if (t < head) p[t] = T{};
  p += head;
  n -= head;
  for (int64_t i = t; i < n / W; i += lanes)
    __stcs(reinterpret_cast<uint4*>(p) + i, make_uint4(0, 0, 0, 0));
  if (t < n % W) p[n / W * W + t] = T{};
}

// A team's share of the columns [blockIdx.y * lanes * VEC, ...) of its items.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embedding_sum_kernel(const SumArgs s) {
  using V = RowVec<T, VEC>;
  constexpr int U = 8;
  const int per = blockDim.x / s.lanes, t = threadIdx.x % s.lanes;
  const int64_t share = (int64_t)blockIdx.x * per + threadIdx.x / s.lanes;
  if (share >= s.shares) return;
  const int64_t items = TOKEN_COST * s.N + s.V;
  const int64_t d0 = share * s.share, d1 = min(items, d0 + s.share);
  int64_t j = tokens_before(s.pairs, s.N, d0);
  const int64_t j1 = tokens_before(s.pairs, s.N, d1);
  // rows whose end lies before d0 and d1 (a place inside a token counts as behind it)
  int64_t v = max(d0 - TOKEN_COST * j, j > 0 ? (int64_t)s.pairs[j - 1].x : 0);
  const int64_t v1 = max(d1 - TOKEN_COST * j1, j1 > 0 ? (int64_t)s.pairs[j1 - 1].x : 0);
  const int64_t c = ((int64_t)blockIdx.y * s.lanes + t) * VEC;
  const bool in = c < s.D;
  // the first row continues one of an earlier share
  bool open = j > 0 && v < s.V && s.pairs[j - 1].x == v;
  if (t == 0 && blockIdx.y == 0) {
    s.flags[share] = (open ? 1 : 0) | (v1 > v ? 2 : 0);
    s.rows[share] = v;
  }
  const T* dout = (const T*)s.dout + c;
  T* dw = (T*)s.dweight + c;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  auto end_row = [&]() {
    if (in) {
      if (open) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) s.head[share * s.D + c + k] = acc[k];
      } else {
        V r;
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] *= s.scale;
        r.set(acc);
        r.store_stream(dw + v * s.D);
      }
    }
    open = false;
    ++v;
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  };
  // row ends up to row `to`: this row's, then absent ones.  Longer runs of those are one
  // range of zeros, of which each column range takes its part (8604 tokens of 132453 rows
  // of 1095 fp32 channels: 222 us against 339 us row by row; runs of two rows lose by it).
  auto end_rows = [&](int64_t to) {
    end_row();
    if (to - v >= 4) {
      const int64_t first = v * s.D, n = (to - v) * s.D;
      const int64_t part = (n + gridDim.y - 1) / gridDim.y, lo = min(n, blockIdx.y * part);
      fill_zeros((T*)s.dweight, first + lo, first + min(n, lo + part), t, s.lanes);
      v = to;
    }
    while (v < to) end_row();
  };
  const int lane = threadIdx.x & 31;
  if constexpr (SUM_ASYNC<T, VEC>) {
    // Each thread copies its own pieces of the rows and reads only those, so that no
    // thread waits for another; the pairs come 32 at a time, a copy for each warp.
    extern __shared__ __align__(16) uint4 s_rows[];      // [SUM_STAGES * SUM_BATCH][blockDim.x]
    __shared__ int2 s_ring[8][64];
    int2* const ring = s_ring[threadIdx.x >> 5];
    V* const rows = reinterpret_cast<V*>(s_rows) + threadIdx.x;
    const int n = (int)(j1 - j);
    const int2* const src = s.pairs + j;
    int2 ahead = lane < n ? __ldg(src + lane) : make_int2(0, 0);
    auto fetch = [&](int i0) {
      if ((i0 & 31) == 0 && i0 < n) {
        __syncwarp();
        ring[(i0 & 63) + lane] = ahead;
        __syncwarp();
        if (i0 + 32 + lane < n) ahead = __ldg(src + i0 + 32 + lane);
      }
#pragma unroll
      for (int u = 0; u < SUM_BATCH; ++u) {
        const int i = i0 + u;
        if (i < n) {
          const int2 p = ring[i & 63];
          if (in && p.x < s.V)
            tp_cp_async16(rows + (i % (SUM_STAGES * SUM_BATCH)) * blockDim.x,
                          dout + (int64_t)p.y * s.D, 16);
        }
      }
      tp_cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < SUM_STAGES - 1; ++k) fetch(k * SUM_BATCH);
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += SUM_BATCH) {
      fetch(i0 + (SUM_STAGES - 1) * SUM_BATCH);
      tp_cp_async_wait<SUM_STAGES - 1>();
#pragma unroll
      for (int u = 0; u < SUM_BATCH; ++u) {
        const int i = i0 + u;
        const int key = i < n ? ring[i & 63].x : (int)s.V;
        if (key >= s.V) break;               // dropped tokens come last
        if (v < key) end_rows(key);
        if (in) {
          const V row = rows[(i % (SUM_STAGES * SUM_BATCH)) * blockDim.x];
          float f[VEC];
          row.get(f);
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += f[k];
        }
      }
    }
  } else {
    // pairs of 128 tokens at a time in shared memory, a copy for each warp
    __shared__ int2 s_pairs[8][SUM_CHUNK];
    int2* const pairs = s_pairs[threadIdx.x >> 5];
    for (; j < j1; j += SUM_CHUNK) {
      const int m = (int)min((int64_t)SUM_CHUNK, j1 - j);
      __syncwarp();
  #pragma unroll
      for (int k = 0; k < SUM_CHUNK / 32; ++k)
        if (k * 32 + lane < m) pairs[k * 32 + lane] = __ldg(s.pairs + j + k * 32 + lane);
      __syncwarp();
  #pragma unroll 1
      for (int i = 0; i < m; i += U) {
        V row[U];
        const int n = min(U, m - i);
  #pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u < n) {
            const int2 p = pairs[i + u];
            if (in && p.x < s.V) row[u].load_stream(dout + (int64_t)p.y * s.D);
          }
        }
  #pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u < n) {
            const int key = pairs[i + u].x;
            if (key >= s.V) break;             // dropped tokens come last
            if (v < key) end_rows(key);
            if (in) {
              float f[VEC];
              row[u].get(f);
  #pragma unroll
              for (int k = 0; k < VEC; ++k) acc[k] += f[k];
            }
          }
        }
      }
    }
  }
  if (v < v1) end_rows(v1);
  if (in) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) s.tail[share * s.D + c + k] = acc[k];
  }
}

// Rows over several shares: the share that ends such a row (its first row is
// open and it has an end) adds the tails of the shares before it, in order,
// and its head.  A block per share; a row over more than 16 shares takes one per
// 256 columns, whose warps add contiguous parts of the shares.
template <typename T>
__global__ void __launch_bounds__(256) embedding_join_kernel(const SumArgs s) {
  const int64_t share = blockIdx.x;
  if (s.flags[share] != 3) return;
  __shared__ int s_first[8];
  __shared__ float s_part[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the share in which the row began: back over shares wholly inside it (flag 1)
  int64_t first = share - 1;
  for (int64_t p0 = share - 1;; p0 -= 256) {
    const int64_t p = p0 - threadIdx.x;
    const bool stop = p <= 0 || s.flags[p] != 1;
    const unsigned any = __ballot_sync(0xffffffffu, stop);
    if (lane == 0) s_first[warp] = any ? warp * 32 + __ffs(any) - 1 : 256;
    __syncthreads();
    int at = 256;
#pragma unroll
    for (int w = 7; w >= 0; --w) at = s_first[w] < 256 ? s_first[w] : at;
    __syncthreads();
    first = p0 - at;
    if (at < 256) break;
  }
  T* const out = (T*)s.dweight + s.rows[share] * s.D;
  const float* const head = s.head + share * s.D;
  RowVec<T, 1> r;
  if (share - first <= 16) {
    if (blockIdx.y > 0) return;
    for (int64_t c = threadIdx.x; c < s.D; c += 256) {
      float t = 0.f;
#pragma unroll 4
      for (int64_t p = first; p < share; ++p) t += s.tail[p * s.D + c];
      t = (t + head[c]) * s.scale;
      r.set(&t);
      r.store(out + c);
    }
    return;
  }
  const int64_t c0 = (int64_t)blockIdx.y * 256;
  const int64_t per = (share - first + 7) / 8;
  const int64_t lo = min(share, first + warp * per), hi = min(share, lo + per);
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
#pragma unroll 4
  for (int64_t p = lo; p < hi; ++p)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + j * 32 + lane < s.D) acc[j] += s.tail[p * s.D + c0 + j * 32 + lane];
#pragma unroll
  for (int j = 0; j < 8; ++j) s_part[warp][j * 32 + lane] = acc[j];
  __syncthreads();
  const int64_t c = c0 + threadIdx.x;
  if (c >= s.D) return;
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += s_part[w][threadIdx.x];
  t = (t + head[c]) * s.scale;
  r.set(&t);
  r.store(out + c);
}

// ---------------------------------------------------------------- positions
// dpos[t] = sum over the sequences of dout[., t], with IDS of the tokens whose id is in
// [0, V).  SPLIT: the block's 8 warps take contiguous ranges of the sequences for 32
// vectors of one position; else each warp has 32 vectors of its own and adds all
// sequences.  (IDS: registers for three blocks an SM, 64 x 1024 x 640 bf16 23 us, against
// 27 with 112 registers and 18 without ids.)
template <typename T, int VEC, bool SPLIT, bool IDS>
__global__ void __launch_bounds__(256, IDS ? 3 : 1) embedding_pos_kernel(int64_t B, int64_t steps, int64_t L,
                                                            int64_t D,
                                                            const T* __restrict__ dout,
                                                            const void* ids, int ids64,
                                                            int64_t V, T* dpos) {
  using R = RowVec<T, VEC>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = SPLIT ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
  const int64_t c = ((int64_t)blockIdx.y * 32 + lane) * VEC;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  const int64_t per = (B + 7) / 8, lo = SPLIT ? warp * per : 0;
  const int64_t hi = SPLIT ? min(B, lo + per) : B;
  // (IDS: lanes behind the row read its first channels, so that the warp stays together)
  if (t < steps && (IDS || c < D)) {
    const T* p = dout + (lo * steps + t) * D + (!IDS || c < D ? c : 0);
    const int n = (int)max(hi - lo, (int64_t)0);      // (B is held below 2^31 - 64)
    // 32 sequences' ids by one load, a lane each, the next ones on their way with the rows
    int64_t at = (lo + lane) * steps + t;
    bool ahead = false;
    auto next_ids = [&](int b) {
      if (b + lane < n) {
        const int64_t id = load_index(ids, ids64, at);
        ahead = id >= 0 && id < V;
      }
      at += 32 * steps;
    };
    if (IDS) next_ids(0);
    unsigned known = ~0u;
    for (int b = 0; b < n; b += 8) {
      R r[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        r[u].zero();
        if (b + u < n) r[u].load(p);
        p += steps * D;
      }
      if (IDS) {
        known >>= 8;
        if ((b & 31) == 0) {
          known = __ballot_sync(0xffffffffu, ahead);
          next_ids(b + 32);
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        float f[VEC];
        r[u].get(f);
        if (b + u < n && (!IDS || ((known >> u) & 1)))
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += f[k];
      }
    }
  }
  if constexpr (SPLIT) {
    __shared__ float s[8][32 * VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[warp][lane * VEC + k] = acc[k];
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += s[w][lane * VEC + k];
      acc[k] = v;
    }
  }
  if (t < L && c < D) {
    R r;
    r.set(acc);
    r.store(dpos + t * D + c);
  }
}

template <typename T, int VEC>
bool vec_ok(int64_t D, std::initializer_list<const void*> ps,
            std::initializer_list<int64_t> strides) {
  const uintptr_t m = sizeof(T) * VEC - 1;
  if (D % VEC) return false;
  for (const void* p : ps)
    if (((uintptr_t)p) & m) return false;
  for (int64_t s : strides)
    if (s % VEC) return false;
  return true;
}

int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }

// Threads of a team: whole warps over the row's vectors, at most 256 a column range.
int sum_lanes(int64_t D, int vec, int64_t* ranges) {
  const int64_t nv = ceil_div(D, (int64_t)vec);
  *ranges = ceil_div(nv, (int64_t)256);
  return (int)(ceil_div(ceil_div(nv, *ranges), (int64_t)32) * 32);
}

// Teams of a block: as many as make 128 threads, at least one.
int sum_teams(int lanes) { return lanes >= 128 ? 1 : 128 / lanes; }

struct SumPlan {
  int64_t share, shares;
};

// As many shares as teams fit at once (768 threads with their 256 bytes of rows on an SM,
// 819 of 80 registers where rows stay in those), so
// that there is one wave of them and each searches its place once; at least 16
// items each, so that partial sums stay few (two or four waves: the sums of 60 x 4096 tokens
// 83, 85 and 92 us, their joins 8, 14 and 25 us).  By the sizes alone, for 16 bytes a
// thread: rows of single channels take the same shares.
SumPlan sum_plan(int64_t N, int64_t V, int64_t D, int esize) {
  const int64_t items = TOKEN_COST * N + V;
  int64_t ranges;
  const int lanes = sum_lanes(D, 16 / esize, &ranges);
  const int per = sum_teams(lanes);
  int64_t teams = (esize == 4 ? 768 : 819) / (lanes * per) * per / ranges;
  if (teams < 1) teams = 1;
  int64_t share = ceil_div(items, num_sms() * teams);
  if (share < 16 * TOKEN_COST) share = 16 * TOKEN_COST;
  return {share, ceil_div(items, share)};
}

struct Workspace {
  int2* pairs[2];
  int *hist, *flags;
  int64_t* rows;
  float *head, *tail;
  int64_t bytes;
};

Workspace layout(int64_t N, int64_t V, int64_t D, int esize, void* base) {
  const SortPlan sp = sort_plan(N, V);
  const SumPlan su = sum_plan(N, V, D, esize);
  Workspace w;
  char* p = (char*)base;
  auto take = [&](int64_t bytes) {
    char* q = p;
    p += round16(bytes);
    return (void*)q;
  };
  for (int k = 0; k < 2; ++k) w.pairs[k] = (int2*)take(N * 8);
  w.hist = (int*)take((int64_t)(sp.cluster ? sp.cluster * sp.passes : sp.tiles) * (4 << sp.bits));
  w.flags = (int*)take(su.shares * 4);
  w.rows = (int64_t*)take(su.shares * 8);
  w.head = (float*)take(su.shares * D * 4);
  w.tail = (float*)take(su.shares * D * 4);
  w.bytes = p - (char*)base;
  return w;
}

// Few tokens: a block per token, so that each row's loads are issued at once.
// Many: a warp takes four rows of up to 64 vectors, or four vectors of a longer
// row, at a time (32 x 4096 tokens of 1024 bf16 channels: 61 us against 70 us with
// four rows; 16 x 2048 of 512: 18 and 15 us).
template <typename T, int VEC>
int fwd_rows(const EmbeddingArgs& a, cudaStream_t stream) {
  const IndexErrorWords bad = index_error_words();
  const bool many = a.N >= 16 * (int64_t)num_sms(), rows = many && a.D / VEC <= 64;
  const int lanes = many ? 32 : 128;
  const int64_t want = ceil_div(a.N, rows ? (int64_t)16 : (many ? (int64_t)4 : (int64_t)1));
  const int64_t cap = (int64_t)num_sms() * 64;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  if (rows) embedding_fwd_kernel<T, VEC, 4, 1><<<grid, 128, 0, stream>>>(a, lanes, bad);
  else embedding_fwd_kernel<T, VEC, 1, 4><<<grid, 128, 0, stream>>>(a, lanes, bad);
  return launch_status();
}

template <typename T>
int fwd(const EmbeddingArgs& a, cudaStream_t stream) {
  constexpr int WIDE = 16 / sizeof(T);
  if (vec_ok<T, WIDE>(a.D, {a.weight, a.pos_weight, a.out}, {a.ldw, a.pos_weight ? a.ldp : 0}))
    return fwd_rows<T, WIDE>(a, stream);
  return fwd_rows<T, 1>(a, stream);
}

template <typename T, int VEC>
int sum(SumArgs s, cudaStream_t stream) {
  int64_t ranges;
  s.lanes = sum_lanes(s.D, VEC, &ranges);
  const int per = sum_teams(s.lanes);
  const int threads = s.lanes * per;
  const dim3 grid((unsigned)ceil_div(s.shares, (int64_t)per), (unsigned)ranges);
  const size_t smem = SUM_ASYNC<T, VEC> ? (size_t)SUM_STAGES * SUM_BATCH * 16 * threads : 0;
  if (smem > 40 * 1024) {
    const int st = allow_smem((const void*)embedding_sum_kernel<T, VEC>, smem);
    if (st != TP_OK) return st;
  }
  embedding_sum_kernel<T, VEC><<<grid, threads, smem, stream>>>(s);
  // (each launch that the next one's indices come from is asked for, so that none runs on
  // what a refused one left in the workspace)
  const int st = launch_status();
  if (st != TP_OK) return st;
  const dim3 join((unsigned)s.shares, (unsigned)ceil_div(s.D, (int64_t)256));
  embedding_join_kernel<T><<<join, 256, 0, stream>>>(s);
  return launch_status();
}

int sort_in_cluster(const SortPlan& p, const Workspace& w, const Keys& keys, int64_t N,
                    cudaStream_t stream) {
  ClusterSortArgs s;
  s.keys = keys;
  for (int k = 0; k < 2; ++k) s.pairs[k] = w.pairs[k];
  s.hist = w.hist;
  s.N = N;
  s.passes = p.passes;
  s.bits = p.bits;
  s.S = p.cluster;
  const size_t smem = sizeof(uint16_t) * SC_WARPS * ((size_t)1 << p.bits);
  const int st = allow_smem((const void*)sort_cluster_kernel, smem);
  if (st != TP_OK) return st;
  if (p.cluster > 8) {
    const cudaError_t e = cudaFuncSetAttribute((const void*)sort_cluster_kernel,
                                               cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return cuda_status(e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.cluster);
  cfg.blockDim = dim3(SC_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)p.cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, sort_cluster_kernel, s));
}

template <typename T>
int sum_any(const SumArgs& s, cudaStream_t stream) {
  constexpr int WIDE = 16 / sizeof(T);
  if (vec_ok<T, WIDE>(s.D, {s.dout, s.dweight}, {})) return sum<T, WIDE>(s, stream);
  return sum<T, 1>(s, stream);
}

struct PosArgs {
  int64_t B, steps, L, D;
  const void *dout, *ids;
  int ids64;
  int64_t V;
  void* dpos;
};

template <typename T, int VEC, bool IDS>
int pos_rows(const PosArgs& a, cudaStream_t stream) {
  const unsigned columns = (unsigned)ceil_div(a.D, (int64_t)32 * VEC);
  // few positions for the GPU, or long sums: the sequences are shared out as well (114
  // sequences of 205 x 1152 fp32: 29 us against 65; 32 of 4096 x 1024 bf16: 59 against 47)
  if (a.B > 8 && a.steps * columns < (a.B > 64 ? 64 : 8) * (int64_t)num_sms())
    embedding_pos_kernel<T, VEC, true, IDS><<<dim3((unsigned)a.L, columns), 256, 0, stream>>>(
        a.B, a.steps, a.L, a.D, (const T*)a.dout, a.ids, a.ids64, a.V, (T*)a.dpos);
  else
    embedding_pos_kernel<T, VEC, false, IDS>
        <<<dim3((unsigned)ceil_div(a.L, (int64_t)8), columns), 256, 0, stream>>>(
            a.B, a.steps, a.L, a.D, (const T*)a.dout, a.ids, a.ids64, a.V, (T*)a.dpos);
  return launch_status();
}

template <typename T, bool IDS>
int pos(const PosArgs& a, cudaStream_t stream) {
  constexpr int WIDE = 16 / sizeof(T);
  if (vec_ok<T, WIDE>(a.D, {a.dout, a.dpos}, {})) return pos_rows<T, WIDE, IDS>(a, stream);
  return pos_rows<T, 1, IDS>(a, stream);
}

}  // namespace

int launch_embedding_fwd(const EmbeddingArgs& a, cudaStream_t stream) {
  return a.dtype == TP_DTYPE_F32 ? fwd<float>(a, stream) : fwd<bf16_t>(a, stream);
}

int64_t embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D) {
  const int64_t a = layout(N, V, D, 4, nullptr).bytes, b = layout(N, V, D, 2, nullptr).bytes;
  return a > b ? a : b;
}

int launch_embedding_bwd(int dtype, int ids64, int64_t N, int64_t D, const void* ids,
                         const void* dout, int64_t V, float scale, int64_t padding_idx,
                         const void* other, int64_t other_rows, void* dweight, void* workspace,
                         cudaStream_t stream) {
  const Keys keys = {ids, other, ids64, V, padding_idx, other_rows};
  const SortPlan p = sort_plan(N, V);
  const int esize = dtype == TP_DTYPE_F32 ? 4 : 2;
  const Workspace w = layout(N, V, D, esize, workspace);
  const int bins = 1 << p.bits;
  const size_t place_smem = sizeof(int) * SORT_WARPS * bins;
  if (place_smem > 48 * 1024) {
    const int st = allow_smem((const void*)sort_place_kernel, place_smem);
    if (st != TP_OK) return st;
  }
  int at = N <= SMALL_TOKENS ? 1 : (p.cluster ? (p.passes & 1) : 0);
  if (N > 0 && N <= SMALL_TOKENS) {
    sort_small_kernel<<<1, (unsigned)SMALL_TOKENS, 0, stream>>>(keys, (int)N, w.pairs[0]);
    const int st = launch_status();
    if (st != TP_OK) return st;
  } else if (p.cluster && N > 0) {
    const int st = sort_in_cluster(p, w, keys, N, stream);
    if (st != TP_OK) return st;
  }
  for (int pass = 0; pass < p.passes && N > SMALL_TOKENS && !p.cluster; ++pass) {
    SortArgs s;
    s.keys = keys;
    s.first = pass == 0;
    s.in = w.pairs[at ^ 1];
    s.out = w.pairs[at];
    s.hist = w.hist;
    s.N = N;
    s.tile = p.tile;
    s.tiles = p.tiles;
    s.shift = pass * p.bits;
    s.bins = bins;
    s.bits = p.bits;
    sort_count_kernel<<<(unsigned)p.tiles, SORT_THREADS, sizeof(int) * bins, stream>>>(s);
    int st = launch_status();
    if (st != TP_OK) return st;
    sort_place_kernel<<<(unsigned)p.tiles, SORT_THREADS, place_smem, stream>>>(s);
    st = launch_status();
    if (st != TP_OK) return st;
    at ^= 1;
  }
  const SumPlan su = sum_plan(N, V, D, esize);
  SumArgs s;
  s.pairs = w.pairs[at ^ 1];
  s.N = N;
  s.V = V;
  s.D = D;
  s.dout = dout;
  s.scale = scale;
  s.dweight = dweight;
  s.share = su.share;
  s.shares = su.shares;
  s.head = w.head;
  s.tail = w.tail;
  s.flags = w.flags;
  s.rows = w.rows;
  return dtype == TP_DTYPE_F32 ? sum_any<float>(s, stream) : sum_any<bf16_t>(s, stream);
}

int launch_embedding_pos_bwd(int dtype, int64_t N, int64_t T, int64_t D, const void* dout,
                             int64_t L, const void* ids, int ids64, int64_t V, void* dpos,
                             cudaStream_t stream) {
  const PosArgs a = {T > 0 ? N / T : 0, T, L, D, dout, ids, ids64, V, dpos};
  if (dtype == TP_DTYPE_F32)
    return ids != nullptr ? pos<float, true>(a, stream) : pos<float, false>(a, stream);
  return ids != nullptr ? pos<bf16_t, true>(a, stream) : pos<bf16_t, false>(a, stream);
}

}  // namespace tp
