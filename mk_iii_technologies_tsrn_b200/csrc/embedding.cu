// embedding.cu -- the token embedding of a language model and its gradient:
//
//   out[i] = weight[id_i] * scale (+ pos_weight[position_i])
//   dweight[v] = scale * sum over i with id_i = v of dout[i]
//
// as `embed(ids) * sqrt(d_model) + pos_embed(positions)` of the token models
// (tropformer_dropin.py:616-720).  An id or position outside its table is
// never read: its row of `out` is NaN, it adds to no gradient, and
// TP_DEVERR_INDEX is recorded in the device error word.
//
// The forward is a row gather: bound by the rows read and written.
//
// The gradient sums rows by token.  Adding them with atomics would make the
// order, and so the bits, depend on timing, and a frequent token would
// serialise; instead the tokens are sorted by id (a stable counting sort, so
// equal ids keep their order) and the sorted rows summed in that order:
//
// 1. sort: the id is cut into one or two digits of at most 11 bits.  Per
//    digit, one kernel counts the digits of each tile of tokens and one
//    places them: each warp ranks its run of tokens 32 at a time by digit
//    match, on top of the counts of earlier bins, tiles and warps.
// 2. sum: tokens and table rows form one list of N + V items (the tokens of a
//    row, then the row's end).  Each team of threads takes an equal share of
//    it, found by bisection, whatever the distribution of the ids: it adds a
//    row of dout per token and writes a row of the gradient (zeros for an
//    absent id) per end.  So every dout row is read once and every gradient
//    row written once: the bytes the result needs.
// 3. join: a table row whose tokens reach over several shares left fp32
//    partial sums in the workspace; they are added in order.
#include <initializer_list>

#include "maxplus_internal.cuh"
#include "rowvec.cuh"

namespace tp {

namespace {

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  return is64 ? __ldg((const long long*)p + i) : (int64_t)__ldg((const int*)p + i);
}

// ---------------------------------------------------------------- forward
template <typename T, int VEC>
__global__ void __launch_bounds__(128) embedding_fwd_kernel(const EmbeddingArgs a, int lanes,
                                                            int* err) {
  using V = RowVec<T, VEC>;
  constexpr int U = 4;
  const int t = threadIdx.x % lanes, per = blockDim.x / lanes;
  const int64_t nv = a.D / VEC;
  for (int64_t i = (int64_t)blockIdx.x * per + threadIdx.x / lanes; i < a.N;
       i += (int64_t)gridDim.x * per) {
    const int64_t id = load_index(a.ids, a.ids64, i);
    int64_t at = 0;
    bool ok = id >= 0 && id < a.V;
    if (a.pos_weight) {
      at = a.positions ? load_index(a.positions, a.ids64, i) : i % a.T;
      ok = ok && at >= 0 && at < a.L;
    }
    if (!ok && t == 0) tp_record_device_error(err, TP_DEVERR_INDEX);
    const T* wr = (const T*)a.weight + (ok ? id * a.ldw : 0);
    const T* pr = a.pos_weight ? (const T*)a.pos_weight + (ok ? at * a.ldp : 0) : nullptr;
    T* o = (T*)a.out + i * a.D;
    for (int64_t v0 = t; v0 < nv; v0 += U * lanes) {
      V w[U], p[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t v = v0 + k * lanes;
        if (ok && v < nv) {
          w[k].load(wr + v * VEC);
          if (pr) p[k].load(pr + v * VEC);
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t v = v0 + k * lanes;
        if (v >= nv) break;
        float f[VEC];
        w[k].get(f);
        if (pr) {
          float q[VEC];
          p[k].get(q);
          // product and sum rounded one by one, as the unfused expression
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] = __fadd_rn(__fmul_rn(f[j], a.scale), q[j]);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] = __fmul_rn(f[j], a.scale);
        }
        if (!ok) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] = __int_as_float(0x7fc00000);
        }
        V r;
        r.set(f);
        r.store(o + v * VEC);
      }
    }
  }
}

// ---------------------------------------------------------------- sort
constexpr int SORT_THREADS = 256;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_MAX_BITS = 11;
constexpr int64_t SORT_MAX_TILES = 128;

struct SortPlan {
  int64_t tile;     // tokens per block, a multiple of 32 * SORT_WARPS
  int tiles;
  int passes, bits; // digits per key, bits per digit
};

SortPlan sort_plan(int64_t N, int64_t V) {
  SortPlan p;
  int bits = 1;
  while (((int64_t)1 << bits) <= V) ++bits;     // keys 0 .. V (V: not in the table)
  p.passes = bits <= SORT_MAX_BITS ? 1 : (bits <= 2 * SORT_MAX_BITS ? 2 : 3);
  p.bits = (bits + p.passes - 1) / p.passes;
  const int64_t unit = 32 * SORT_WARPS;
  p.tile = 8 * unit;                            // 2048 tokens
  if (ceil_div(N, p.tile) > SORT_MAX_TILES)
    p.tile = ceil_div(ceil_div(N, SORT_MAX_TILES), unit) * unit;
  p.tiles = (int)ceil_div(N, p.tile);
  return p;
}

struct SortArgs {
  const void* ids;        // first pass: the caller's ids
  int ids64;
  int64_t V, padding_idx;
  const int* keys_in;     // later passes: keys and token numbers of the pass before
  const int* toks_in;
  int* keys_out;
  int* toks_out;
  int* hist;              // [tiles][bins]
  int64_t N, tile;
  int tiles, shift, bins;
  int first;
};

__device__ __forceinline__ int sort_key(const SortArgs& s, int64_t i) {
  if (!s.first) return s.keys_in[i];
  const int64_t id = load_index(s.ids, s.ids64, i);
  return (id < 0 || id >= s.V || id == s.padding_idx) ? (int)s.V : (int)id;
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
      if (s.tiles == 1) {
#pragma unroll
        for (int w = 0; w < SORT_WARPS; ++w) all += s_mem[w * s.bins + b];
      } else {
#pragma unroll 8
        for (int t = 0; t < s.tiles; ++t) {
          const int n = s.hist[(int64_t)t * s.bins + b];
          all += n;
          if (t < (int)blockIdx.x) earlier += n;
        }
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
    const int d = in ? (key >> s.shift) & (s.bins - 1) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, d);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int at = 0;
    if (in) at = mine[d] + rank;
    __syncwarp();
    if (in) {
      if (rank == 0) mine[d] += __popc(same);
      s.keys_out[at] = key;
      s.toks_out[at] = s.first ? (int)i : s.toks_in[i];
    }
    __syncwarp();
  }
}

// ---------------------------------------------------------------- sum
struct SumArgs {
  const int* keys;      // sorted; V: dropped
  const int* toks;
  int64_t N, V, D;
  const void* dout;
  float scale;
  void* dweight;
  int64_t share;        // items per team
  int64_t shares;
  int lanes;            // threads of a team
  float* head;          // [shares][D]: end of a row begun in an earlier share
  float* tail;          // [shares][D]: begin of a row that ends in a later share
  int* flags;           // [shares]: bit 0 the first row began earlier, bit 1 an end lies inside
};

// Tokens among the first `d` items of the list (the tokens of row 0, the end of
// row 0, the tokens of row 1, ...): the smallest j with keys[j] + j >= d, as
// token j is item keys[j] + j.
__device__ __forceinline__ int64_t tokens_before(const int* keys, int64_t N, int64_t d) {
  int64_t lo = 0, hi = min(N, d);
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if ((int64_t)__ldg(keys + mid) + mid >= d) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// A team's share of the columns [blockIdx.y * lanes * VEC, ...) of its items.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embedding_sum_kernel(const SumArgs s) {
  using V = RowVec<T, VEC>;
  constexpr int U = 8;
  const int per = blockDim.x / s.lanes, t = threadIdx.x % s.lanes;
  const int64_t share = (int64_t)blockIdx.x * per + threadIdx.x / s.lanes;
  if (share >= s.shares) return;
  const int64_t items = s.N + s.V;
  const int64_t d0 = share * s.share, d1 = min(items, d0 + s.share);
  int64_t j = tokens_before(s.keys, s.N, d0);
  const int64_t j1 = tokens_before(s.keys, s.N, d1);
  int64_t v = d0 - j;
  const int64_t v1 = d1 - j1;          // rows whose end lies before d1
  const int64_t c = ((int64_t)blockIdx.y * s.lanes + t) * VEC;
  const bool in = c < s.D;
  // the first row continues one of an earlier share
  bool open = j > 0 && v < s.V && s.keys[j - 1] == v;
  if (t == 0 && blockIdx.y == 0) s.flags[share] = (open ? 1 : 0) | (v1 > v ? 2 : 0);
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
  while (j < j1) {
    V row[U];
    int key[U];
    const int n = (int)min((int64_t)U, j1 - j);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < n) {
        key[u] = __ldg(s.keys + j + u);
        if (in && key[u] < s.V) row[u].load_stream(dout + (int64_t)__ldg(s.toks + j + u) * s.D);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < n && key[u] < s.V) {
        while (v < key[u]) end_row();
        if (in) {
          float f[VEC];
          row[u].get(f);
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += f[k];
        }
      }
    }
    j += n;
  }
  while (v < v1) end_row();
  if (in) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) s.tail[share * s.D + c + k] = acc[k];
  }
}

// Rows over several shares: the share that ends such a row (its first row is
// open and it has an end) adds the tails of the shares before it, in order,
// and its head.
template <typename T>
__global__ void __launch_bounds__(128) embedding_join_kernel(const SumArgs s) {
  const int64_t share = blockIdx.x;
  if (s.flags[share] != 3) return;
  __shared__ long long s_first;
  if (threadIdx.x == 0) {
    int64_t p = share - 1;
    while (p > 0 && s.flags[p] == 1) --p;     // shares wholly inside the row
    s_first = p;
  }
  __syncthreads();
  const int64_t first = s_first;
  const int64_t j = tokens_before(s.keys, s.N, share * s.share);
  const int64_t v = share * s.share - j;
  for (int64_t c = threadIdx.x; c < s.D; c += blockDim.x) {
    float acc = 0.f;
#pragma unroll 8
    for (int64_t p = first; p < share; ++p) acc += s.tail[p * s.D + c];
    acc = (acc + s.head[share * s.D + c]) * s.scale;
    RowVec<T, 1> r;
    r.set(&acc);
    r.store((T*)s.dweight + v * s.D + c);
  }
}

// ---------------------------------------------------------------- positions
// dpos[t] = sum over the sequences of dout[., t]: 8 warps take contiguous
// ranges of the sequences for 32 vectors of one position.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embedding_pos_kernel(int64_t B, int64_t steps, int64_t D,
                                                            const T* __restrict__ dout, T* dpos) {
  using V = RowVec<T, VEC>;
  __shared__ float s[8][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x;
  const int64_t c = ((int64_t)blockIdx.y * 32 + lane) * VEC;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  if (t < steps && c < D) {
    const int64_t per = (B + 7) / 8, lo = warp * per, hi = min(B, lo + per);
#pragma unroll 4
    for (int64_t b = lo; b < hi; ++b) {
      V r;
      float f[VEC];
      r.load(dout + (b * steps + t) * D + c);
      r.get(f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += f[k];
    }
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) s[warp][lane * VEC + k] = acc[k];
  __syncthreads();
  if (warp == 0 && c < D) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += s[w][lane * VEC + k];
      acc[k] = v;
    }
    V r;
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

struct SumPlan {
  int64_t share, shares;
};

// About twelve shares per SM (teams that wait on loads overlap), at least 16
// items each so that partial sums stay few.
SumPlan sum_plan(int64_t N, int64_t V) {
  const int64_t items = N + V;
  const int64_t want = (int64_t)num_sms() * 12;
  int64_t share = ceil_div(items, want);
  if (share < 16) share = 16;
  return {share, ceil_div(items, share)};
}

struct Workspace {
  int *keys[2], *toks[2], *hist, *flags;
  float *head, *tail;
  int64_t bytes;
};

Workspace layout(int64_t N, int64_t V, int64_t D, void* base) {
  const SortPlan sp = sort_plan(N, V);
  const SumPlan su = sum_plan(N, V);
  Workspace w;
  char* p = (char*)base;
  auto take = [&](int64_t bytes) {
    char* q = p;
    p += round16(bytes);
    return (void*)q;
  };
  for (int k = 0; k < 2; ++k) {
    w.keys[k] = (int*)take(N * 4);
    w.toks[k] = (int*)take(N * 4);
  }
  w.hist = (int*)take((int64_t)sp.tiles * (4 << sp.bits));
  w.flags = (int*)take(su.shares * 4);
  w.head = (float*)take(su.shares * D * 4);
  w.tail = (float*)take(su.shares * D * 4);
  w.bytes = p - (char*)base;
  return w;
}

template <typename T>
int fwd(const EmbeddingArgs& a, cudaStream_t stream) {
  int* err = device_error_ptr();
  // a warp per token; few tokens: a block per token, so that each row's loads
  // are issued at once
  const int lanes = a.N >= 8 * (int64_t)num_sms() ? 32 : 128;
  const int64_t want = ceil_div(a.N, (int64_t)(128 / lanes)), cap = (int64_t)num_sms() * 64;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  constexpr int WIDE = 16 / sizeof(T);
  if (vec_ok<T, WIDE>(a.D, {a.weight, a.pos_weight, a.out}, {a.ldw, a.pos_weight ? a.ldp : 0}))
    embedding_fwd_kernel<T, WIDE><<<grid, 128, 0, stream>>>(a, lanes, err);
  else
    embedding_fwd_kernel<T, 1><<<grid, 128, 0, stream>>>(a, lanes, err);
  return launch_status();
}

template <typename T, int VEC>
int sum(SumArgs s, cudaStream_t stream) {
  const int64_t nv = ceil_div(s.D, (int64_t)VEC);
  // whole warps over the row's vectors, at most 256 threads a column range
  const int64_t ranges = ceil_div(nv, (int64_t)256);
  s.lanes = (int)(ceil_div(ceil_div(nv, ranges), (int64_t)32) * 32);
  const int per = s.lanes >= 128 ? 1 : 128 / s.lanes;
  const int threads = s.lanes * per;
  const dim3 grid((unsigned)ceil_div(s.shares, (int64_t)per), (unsigned)ranges);
  embedding_sum_kernel<T, VEC><<<grid, threads, 0, stream>>>(s);
  embedding_join_kernel<T><<<(unsigned)s.shares, 128, 0, stream>>>(s);
  return launch_status();
}

template <typename T>
int sum_any(const SumArgs& s, cudaStream_t stream) {
  constexpr int WIDE = 16 / sizeof(T);
  if (vec_ok<T, WIDE>(s.D, {s.dout, s.dweight}, {})) return sum<T, WIDE>(s, stream);
  return sum<T, 1>(s, stream);
}

template <typename T>
int pos(int64_t N, int64_t steps, int64_t D, const void* dout, int64_t L, void* dpos,
        cudaStream_t stream) {
  constexpr int WIDE = 16 / sizeof(T);
  const int64_t B = steps > 0 ? N / steps : 0;
  if (vec_ok<T, WIDE>(D, {dout, dpos}, {}))
    embedding_pos_kernel<T, WIDE><<<dim3((unsigned)L, (unsigned)ceil_div(D, (int64_t)32 * WIDE)),
                                    256, 0, stream>>>(B, steps, D, (const T*)dout, (T*)dpos);
  else
    embedding_pos_kernel<T, 1><<<dim3((unsigned)L, (unsigned)ceil_div(D, (int64_t)32)), 256, 0,
                                 stream>>>(B, steps, D, (const T*)dout, (T*)dpos);
  return launch_status();
}

}  // namespace

int launch_embedding_fwd(const EmbeddingArgs& a, cudaStream_t stream) {
  return a.dtype == TP_DTYPE_F32 ? fwd<float>(a, stream) : fwd<bf16_t>(a, stream);
}

int64_t embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D) {
  return layout(N, V, D, nullptr).bytes;
}

int launch_embedding_bwd(int dtype, int ids64, int64_t N, int64_t D, const void* ids,
                         const void* dout, int64_t V, float scale, int64_t padding_idx,
                         void* dweight, void* workspace, cudaStream_t stream) {
  const SortPlan p = sort_plan(N, V);
  const Workspace w = layout(N, V, D, workspace);
  const int bins = 1 << p.bits;
  const size_t place_smem = sizeof(int) * SORT_WARPS * bins;
  if (place_smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute((const void*)sort_place_kernel,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)place_smem);
    if (e != cudaSuccess) return cuda_status(e);
  }
  int at = 0;
  for (int pass = 0; pass < p.passes && N > 0; ++pass) {
    SortArgs s;
    s.ids = ids;
    s.ids64 = ids64;
    s.V = V;
    s.padding_idx = padding_idx;
    s.first = pass == 0;
    s.keys_in = w.keys[at ^ 1];
    s.toks_in = w.toks[at ^ 1];
    s.keys_out = w.keys[at];
    s.toks_out = w.toks[at];
    s.hist = w.hist;
    s.N = N;
    s.tile = p.tile;
    s.tiles = p.tiles;
    s.shift = pass * p.bits;
    s.bins = bins;
    if (p.tiles > 1)
      sort_count_kernel<<<(unsigned)p.tiles, SORT_THREADS, sizeof(int) * bins, stream>>>(s);
    sort_place_kernel<<<(unsigned)p.tiles, SORT_THREADS, place_smem, stream>>>(s);
    at ^= 1;
  }
  const SumPlan su = sum_plan(N, V);
  SumArgs s;
  s.keys = w.keys[at ^ 1];
  s.toks = w.toks[at ^ 1];
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
  return dtype == TP_DTYPE_F32 ? sum_any<float>(s, stream) : sum_any<bf16_t>(s, stream);
}

int launch_embedding_pos_bwd(int dtype, int64_t N, int64_t T, int64_t D, const void* dout,
                             int64_t L, void* dpos, cudaStream_t stream) {
  return dtype == TP_DTYPE_F32 ? pos<float>(N, T, D, dout, L, dpos, stream)
                               : pos<bf16_t>(N, T, D, dout, L, dpos, stream);
}

}  // namespace tp
