// paged_attention.cuh -- attention of one new token per sequence over a paged key-value
// cache (paged_attention_{f32,bf16}.cu launch it):
//
//   s_j = scale / tau * ((1 - g) q . k_j + g max_f(q_f + k_jf))      (without gate: q . k_j)
//   o   = sum_j softmax(s)_j v_j,  j < lengths[b]
//
// the decoding form of the blended score of the tropical attention modules
// (tropformer_dropin.py:236-260) with grouped query heads.
//
// Every byte of K and V is read once and used for up to 4 (8) query heads: bound by DRAM.
//
// The work is cut into tiles of a few slots.  The tiles of all sequences form one list, in order,
// cut into equal runs whatever the lengths; a warp takes one run for one key head (with a block
// of its query heads), so that the warps of a run, next to one another in the grid, read the same
// slots at the same time: the heads of a slot lie next to one another too.  What a warp finds of a
// sequence is a segment: softmax statistics (maximum and sum, base 2) and sums over V in fp32,
// written out; a second kernel joins the segments of each sequence and head, stores the new token
// and adds the weights to `mass`.  (A block per row and split of its length instead: 4 us of every
// block went into its beginning and end, 237 us where this takes 197.)
//
// Rows come through asynchronous copies into shared memory, STAGES - 1 tiles ahead and
// across the ends of sequences.  The ring begins on 128 bytes: pieces whose place in shared memory
// begins inside 32 bytes are fetched twice from the L2 (16-byte places: 5.4 TB/s for the copies
// alone instead of 7.1).
//
// Measured: 48 sequences of 4096 to 8192 slots of 8 key heads of 128 bf16 channels, 4 query heads
// each, 197 us for 1.22 GB (6.2 TB/s, 94 % of the card's copy rate).
#pragma once

#include <algorithm>

#include "decode.cuh"

namespace tp {

namespace {

__device__ __forceinline__ float neg_inf() { return -__int_as_float(0x7f800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fc00000); }

template <typename T>
struct Chunk;                                  // 16 bytes of a row as floats
template <>
struct Chunk<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
};
template <>
struct Chunk<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};

__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(uint16_t* p, float v) {
  *p = __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

__device__ __forceinline__ const char* shfl_ptr(const char* p, int lane) {
  return (const char*)__shfl_sync(0xffffffffu, (unsigned long long)p, lane);
}

// 16 bytes copied to shared memory, at constant offsets from both addresses
template <int TO, int FROM>
__device__ __forceinline__ void copy16(uint32_t to, const char* from) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(to), "l"(from), "n"(TO),
               "n"(FROM)
               : "memory");
}

// The slots in use of sequence b (0 where the length is none, or the pages are not there).
__device__ __forceinline__ int slots_of(const PagedAttentionArgs& a, int b) {
  const int n = __ldg(a.lengths + b);
  return n < 0 || n > a.capacity || a.c.pages == 0 ? 0 : n;
}

// ---------------------------------------------------------------- the warps' runs of tiles
// A tile of the list.
struct Place {
  int b, tile, tiles, n;      // n: slots in use
};

// On to the next tile; behind the last sequence n is left as it was.
template <int TK>
__device__ __forceinline__ void forward(const PagedAttentionArgs& a, Place& p) {
  if (++p.tile < p.tiles) return;
  p.tile = 0;
  int n = 0;
  while (++p.b < a.B && (n = slots_of(a, p.b)) == 0) {
  }
  if (n > 0) {
    p.n = n;
    p.tiles = (n + TK - 1) / TK;
  }
}

// The first tile of run `run`, and how many there are.  Block 0 notes the runs of each sequence
// for the second kernel.
template <int TK>
__device__ __forceinline__ Place place_of_run(const PagedAttentionArgs& a, int run, int& count) {
  __shared__ int64_t starts[ATT_WARPS * 32 + 1];
  __shared__ int64_t sums[ATT_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + ATT_WARPS * 32 - 1) / (ATT_WARPS * 32);
  const int from = min(a.B, tid * per), to = min(a.B, from + per);
  int64_t mine = 0;
  for (int b = from; b < to; ++b) mine += (slots_of(a, b) + TK - 1) / TK;
  int64_t at = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t y = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += y;
  }
  if (lane == 31) sums[warp] = at;
  __syncthreads();
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < ATT_WARPS; ++w) {
    if (w < warp) at += sums[w];
    all += sums[w];
  }
  starts[tid] = at - mine;
  __syncthreads();
  const int64_t runs = min((int64_t)a.runs, all);
  if (blockIdx.x == 0) {                   // the last run that begins at or before a tile has it
    int64_t x = at - mine;
    for (int b = from; b < to; ++b) {
      const int tiles = (slots_of(a, b) + TK - 1) / TK;
      if (tiles == 0) continue;
      const int r0 = (int)(((x + 1) * runs - 1) / all);
      x += tiles;
      a.runs_of[b] = make_int2(r0, (int)((x * runs - 1) / all) - r0 + 1);
    }
  }
  Place p{0, 0, 1, 0};
  count = 0;
  if (run >= runs) return p;
  const int64_t first = run * all / runs;
  count = (int)((run + 1) * all / runs - first);
  // the last thread whose sequences begin at or before it, then the sequence
  int thread = -1;
#pragma unroll
  for (int k = 0; k < ATT_WARPS; ++k)
    thread += __popc(__ballot_sync(0xffffffffu, starts[k * 32 + lane] <= first));
  int64_t x = starts[thread];
  for (p.b = thread * per;; ++p.b) {
    p.n = slots_of(a, p.b);
    p.tiles = (p.n + TK - 1) / TK;
    if (first < x + p.tiles) break;
    x += p.tiles;
  }
  p.tile = (int)(first - x);
  return p;
}

// Where the segment of a run in sequence b is kept, for key head and block of query heads `sub`:
// both only grow along the list, so their sum is another one for every segment.
__device__ __forceinline__ int64_t segment(const PagedAttentionArgs& a, int b, int64_t run, int sub) {
  return (b + run) * (a.c.heads * a.head_blocks) + sub;
}

// A row of NaN: what a page outside the cache holds.
#define TP_NANS_8 0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu
#define TP_NANS_64 TP_NANS_8, TP_NANS_8, TP_NANS_8, TP_NANS_8, TP_NANS_8, TP_NANS_8, TP_NANS_8, TP_NANS_8
__device__ __align__(16) const uint32_t nan_row[256] = {TP_NANS_64, TP_NANS_64, TP_NANS_64, TP_NANS_64};
// What is multiplied with the weight 0 of a slot behind the last one.
__device__ __align__(16) const uint32_t zero_row[256] = {};

// The rows of K and V that a warp copies: each lane knows one slot of a tile.  Slots behind the
// last one have its keys, for scores that are not used, and zeros for values (an infinity of the
// last slot's, times their weight of 0, would be NaN).  The page is asked for one tile before it is
// needed.
template <typename T, int TK>
struct TileRows {
  const PagedAttentionArgs& a;
  const int kvh;
  int page, slot, whole;               // whole: tiles without the new token or a slot too many
  const unsigned pages;
  const bool halves, same;             // half a tile is in one page; K and V are strided alike
  __device__ __forceinline__ TileRows(const PagedAttentionArgs& args, int key_head)
      : a(args), kvh(key_head), page(0), slot(0), whole(0),
        pages((unsigned)min(args.c.pages, (int64_t)INT32_MAX)), halves(args.c.page_size % (TK / 2) == 0),
        same(args.c.k_page == args.c.v_page && args.c.k_slot == args.c.v_slot) {}
  __device__ __forceinline__ void ask(const Place& p) {
    whole = (p.n - (a.key != nullptr)) / TK;
    slot = min(p.tile * TK + ((int)threadIdx.x & (TK - 1)), p.n - 1);
    page = __ldg(a.c.table + (int64_t)p.b * a.c.table_row + a.c.column(slot));
  }
  // Whether each half of the tile is in one page, and no slot of it the new token's or behind the
  // last one; then where the half's first slot lies behind slot 0 of page 0.
  __device__ __forceinline__ bool in_halves(const Place& p) const {
    return __all_sync(0xffffffffu, halves && p.tile < whole && (unsigned)page < pages);
  }
  __device__ __forceinline__ void half_at(const Place& p, int half, int64_t& k_at, int64_t& v_at) const {
    const int first = p.tile * TK + half * (TK / 2), in = a.c.within(first, a.c.column(first));
    const int64_t its = __shfl_sync(0xffffffffu, page, half * (TK / 2));
    k_at = its * a.c.k_page + in * a.c.k_slot;
    v_at = same ? k_at : its * a.c.v_page + in * a.c.v_slot;
  }
  __device__ __forceinline__ void get(const Place& p, const char*& kp, const char*& vp) {
    const int in = a.c.within(slot, a.c.column(slot));
    if (page < 0 || page >= a.c.pages) {
      tp_record_index_error(a.bad.error, a.bad.seen);
      kp = vp = (const char*)nan_row;
      return;
    }
    kp = a.c.k + (int64_t)kvh * a.c.k_head + (int64_t)page * a.c.k_page + (int64_t)in * a.c.k_slot;
    vp = a.c.v + (int64_t)kvh * a.c.v_head + (int64_t)page * a.c.v_page + (int64_t)in * a.c.v_slot;
    if (a.key != nullptr && slot == p.n - 1) {
      kp = (const char*)((const T*)a.key + (int64_t)p.b * a.key_sb + (int64_t)kvh * a.key_sh);
      vp = (const char*)((const T*)a.value + (int64_t)p.b * a.value_sb + (int64_t)kvh * a.value_sh);
    }
    if (p.tile * TK + ((int)threadIdx.x & (TK - 1)) >= p.n) vp = (const char*)zero_row;
  }
};

// ---------------------------------------------------------------- on the CUDA cores
// A slot's channels lie over LPK lanes, 16 bytes each, so that a load instruction of the warp
// reads 32 / LPK whole rows; eight such steps make a tile (4 KB of K and 4 KB of V a chunk).  The
// eight partial sums of a lane are joined over the lanes by halves (4 + 2 + 1 shuffles for eight
// sums), which leaves each lane a slot's score.
constexpr int ATT_STEPS = 8;

__device__ __forceinline__ int reversed3(int i) {
  return ((i & 1) << 2) | (i & 2) | ((i >> 2) & 1);
}

// x[i] of every lane summed (or maximised) over each group of LPK lanes: lane c of a group
// ends with the whole of step reversed3(c & 7).
template <int LPK, typename F>
__device__ __forceinline__ float join_steps(float (&x)[ATT_STEPS], int lane, F op) {
#pragma unroll
  for (int o = 1, n = ATT_STEPS / 2; n >= 1; o *= 2, n /= 2) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? x[i] : x[i + n], keep = up ? x[i + n] : x[i];
      x[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
  float r = x[0];
#pragma unroll
  for (int o = ATT_STEPS; o < LPK; o *= 2) r = op(r, __shfl_xor_sync(0xffffffffu, r, o));
  return r;
}

// A step's chunks of a slot's row, of the lanes that have any.
template <int NCH, int LPK>
__device__ __forceinline__ void copy_chunks(uint32_t to, const char* p, int step, const int (&valid)[NCH]) {
  to += step * NCH * 512;
  if (valid[0] > 0) copy16<0, 0>(to, p);
  if constexpr (NCH > 1)
    if (valid[1] > 0) copy16<512, LPK * 16>(to, p);
}

// T: float, or uint16_t for bf16.  LPK lanes of a slot with NCH chunks of 16 bytes each; G
// query heads at a time; VEC: every row begins and ends on 16 bytes.
template <typename T, int LPK, int NCH, int G, bool GATED, bool VEC, int STAGES>
__global__ void __launch_bounds__(ATT_WARPS * 32) paged_attend_kernel(const PagedAttentionArgs a) {
  constexpr int N = Chunk<T>::N, N2 = N / 2;
  constexpr int KPL = 32 / LPK;                       // slots of a load
  constexpr int TK = ATT_STEPS * KPL;                 // slots of a tile
  constexpr int STAGE = 2 * ATT_STEPS * NCH * 32;     // 16-byte pieces of a warp's stage
  extern __shared__ __align__(128) char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / LPK, c = lane % LPK;
  const int D = a.c.channels, subs = a.c.heads * a.head_blocks;
  const int64_t mine = (int64_t)blockIdx.x * ATT_WARPS + warp;
  const int run = (int)(mine / subs), hsub = (int)(mine - (int64_t)run * subs);
  const int kvh = hsub / a.head_blocks, hblk = hsub - kvh * a.head_blocks;
  int count;
  Place at = place_of_run<TK>(a, run, count);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (count == 0) return;

  uint4* const ring = (uint4*)smem + (size_t)warp * STAGES * STAGE + lane;
  int valid[NCH];              // channels of this lane's chunks
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    valid[ch] = max(0, min(N, D - (c + ch * LPK) * N));
    if (VEC && valid[ch] == 0)         // channels that are not there: zeros, never copied to
      for (int i = ch; i < STAGES * STAGE / 32; i += NCH) ring[i * 32] = make_uint4(0, 0, 0, 0);
  }

  Place ahead = at;
  TileRows<T, TK> rows(a, kvh);
  rows.ask(ahead);
  // (this lane's piece of its first row in page 0, and from one of its rows to the next)
  const int64_t k_step = KPL * a.c.k_slot, v_step = KPL * a.c.v_slot;
  const char* const kmine = a.c.k + (int64_t)kvh * a.c.k_head + sub * a.c.k_slot + c * 16;
  const char* const vmine = a.c.v + (int64_t)kvh * a.c.v_head + sub * a.c.v_slot + c * 16;
  auto issue = [&](int i) {
    if (i < count) {
      const char *kp, *vp;
      uint4* const dst = ring + (size_t)(i % STAGES) * STAGE;
      const uint32_t to = tp_smem_addr(dst);
      const char* from[2 * ATT_STEPS];                        // K, then V
      if (rows.in_halves(ahead)) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          int64_t k_at, v_at;
          rows.half_at(ahead, half, k_at, v_at);
          kp = kmine + k_at;
          vp = vmine + v_at;
#pragma unroll
          for (int step = half * ATT_STEPS / 2; step < (half + 1) * ATT_STEPS / 2; ++step, kp += k_step, vp += v_step) {
            from[step] = kp;
            from[ATT_STEPS + step] = vp;
          }
        }
      } else {
        rows.get(ahead, kp, vp);
#pragma unroll
        for (int step = 0; step < 2 * ATT_STEPS; ++step)
          from[step] = shfl_ptr(step < ATT_STEPS ? kp : vp, step % ATT_STEPS * KPL + sub) + c * 16;
      }
#pragma unroll
      for (int step = 0; step < 2 * ATT_STEPS; ++step) {
        const char* p = from[step];
        if constexpr (VEC) {
          copy_chunks<NCH, LPK>(to, p, step, valid);
        } else {
#pragma unroll
          for (int ch = 0; ch < NCH; ++ch) {
            alignas(16) T e[N];
#pragma unroll
            for (int x = 0; x < N; ++x) e[x] = x < valid[ch] ? *((const T*)(p + ch * LPK * 16) + x) : T(0);
            dst[(step * NCH + ch) * 32] = *(const uint4*)e;
          }
        }
      }
      if (i + 1 < count) {
        forward<TK>(a, ahead);
        rows.ask(ahead);
      }
    }
    tp_cp_async_commit();
  };

  float2 q[G][NCH][N2];                // the query's channels of this lane
  float factor[G], blend[G];
  int h_of[G];
  float m[G], l[G];
  float2 acc[G][NCH][N2];
  auto begin_row = [&]() {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int in_group = hblk * G + g;
      const bool there = in_group < a.group;
      const int h = kvh * a.group + (there ? in_group : 0);
      h_of[g] = there ? h : -1;
      const T* src = (const T*)a.q + (int64_t)at.b * a.q_sb + (int64_t)h * a.q_sh;
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        float e[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
          e[i] = there && i < valid[ch] ? tp_load_as_f32<T>(src + (c + ch * LPK) * N + i) : 0.0f;
#pragma unroll
        for (int i = 0; i < N2; ++i) {
          q[g][ch][i] = make_float2(e[2 * i], e[2 * i + 1]);
          acc[g][ch][i] = make_float2(0.0f, 0.0f);
        }
      }
      factor[g] = (a.tau ? a.scale / __ldg(a.tau + h) : a.scale) * 1.4426950408889634f;
      blend[g] = GATED ? __ldg(a.gate + (int64_t)at.b * a.H + h) : 0.0f;
      m[g] = neg_inf();
      l[g] = 0.0f;
    }
  };
  auto end_row = [&]() {               // the segment, summed over the lanes
    const int64_t seg = segment(a, at.b, run, hsub);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float sum = c < 8 ? l[g] : 0.0f;
#pragma unroll
      for (int o = 1; o < 32; o *= 2)
        if (o < 8 || o >= LPK) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        float* const to = a.part + (seg * G + g) * D + (c + ch * LPK) * N;
#pragma unroll
        for (int x = 0; x < N2; ++x) {
          float2 v = acc[g][ch][x];
#pragma unroll
          for (int o = LPK; o < 32; o *= 2) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
          }
          if (sub == 0 && 2 * x < valid[ch]) to[2 * x] = v.x;
          if (sub == 0 && 2 * x + 1 < valid[ch]) to[2 * x + 1] = v.y;
        }
      }
      if (lane == 0) a.ml[seg * G + g] = make_float2(m[g], sum);
    }
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i);
  bool fresh = true;
  for (int i = 0; i < count; ++i) {
    issue(i + STAGES - 1);
    if (fresh) begin_row();
    tp_cp_async_wait<STAGES - 1>();
    const uint4* kst = ring + (size_t)(i % STAGES) * STAGE;
    const uint4* vst = kst + ATT_STEPS * NCH * 32;

    float dot[G][ATT_STEPS], trop[GATED ? G : 1][ATT_STEPS];
#pragma unroll
    for (int step = 0; step < ATT_STEPS; ++step) {
      float2 d[G];
      float t[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        d[g] = make_float2(0.0f, 0.0f);
        t[g] = neg_inf();
      }
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        float2 k[N2];
        Chunk<T>::unpack(kst[(step * NCH + ch) * 32], k);
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
          for (int x = 0; x < N2; ++x) d[g] = tp_fma2(q[g][ch][x], k[x], d[g]);
          if constexpr (GATED) {
#pragma unroll
            for (int x = 0; x < N2; ++x) {
              const float2 s = tp_add2(q[g][ch][x], k[x]);
              if constexpr (VEC) {
                if (valid[ch] > 0) t[g] = tp_max3_nan(t[g], s.x, s.y);
              } else {
                if (2 * x < valid[ch]) t[g] = tp_max_nan(t[g], s.x);
                if (2 * x + 1 < valid[ch]) t[g] = tp_max_nan(t[g], s.y);
              }
            }
          }
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        dot[g][step] = d[g].x + d[g].y;
        if constexpr (GATED) trop[g][step] = t[g];
      }
    }

    const int key = at.tile * TK + reversed3(c & 7) * KPL + sub;
    float p[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float s = join_steps<LPK>(dot[g], lane, [](float x, float y) { return x + y; });
      if constexpr (GATED) {
        const float t = join_steps<LPK>(trop[g], lane, [](float x, float y) { return tp_max_nan(x, y); });
        s = blend[g] * t + (1.0f - blend[g]) * s;
      }
      s = key < at.n ? s * factor[g] : neg_inf();
      if (a.scores != nullptr && c < 8 && key < at.n && h_of[g] >= 0)
        a.scores[((int64_t)at.b * a.H + h_of[g]) * a.score_row + key] = s;
      float top = s;
#pragma unroll
      for (int o = 1; o < 32; o *= 2)
        if (o < 8 || o >= LPK) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float to = fmaxf(m[g], top);
      const float base = to == neg_inf() ? 0.0f : to;
      if (to != m[g]) {                               // the same for the whole warp
        const float less = tp_ex2(m[g] - base);
        l[g] *= less;
        const float2 both = make_float2(less, less);
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
          for (int x = 0; x < N2; ++x) acc[g][ch][x] = tp_mul2(acc[g][ch][x], both);
        m[g] = to;
      }
      p[g] = tp_ex2(s - base);
      l[g] += p[g];
    }
#pragma unroll
    for (int step = 0; step < ATT_STEPS; ++step) {
      float2 w[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float x = __shfl_sync(0xffffffffu, p[g], sub * LPK + reversed3(step));
        w[g] = make_float2(x, x);
      }
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        float2 v[N2];
        Chunk<T>::unpack(vst[(step * NCH + ch) * 32], v);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int x = 0; x < N2; ++x) acc[g][ch][x] = tp_fma2(w[g], v[x], acc[g][ch][x]);
      }
    }
    fresh = at.tile + 1 == at.tiles || i + 1 == count;
    if (fresh) end_row();
    if (i + 1 < count) forward<TK>(a, at);
  }
  tp_cp_async_wait<0>();
}

// ---------------------------------------------------------------- the rows joined
// (maximum, sum) over the segments of a head, the same in every lane; the loads of 256 segments
// under way together
__device__ __forceinline__ float2 whole_row(const float2* ml, int64_t stride, int parts) {
  const int lane = threadIdx.x & 31;
  float top = neg_inf(), all = 0.0f;
  for (int s0 = 0; s0 < parts; s0 += 256) {
    float2 x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = s0 + 32 * k + lane;
      x[k] = s < parts ? ml[s * stride] : make_float2(neg_inf(), 0.0f);
    }
    float most = top;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = fmaxf(most, x[k].x);
    // (a segment without a maximum counts by its sum, 0 or NaN)
    all = top == neg_inf() ? all : all * tp_ex2(top - most);
#pragma unroll
    for (int k = 0; k < 8; ++k) all += x[k].y * (x[k].x == neg_inf() ? 0.0f : tp_ex2(x[k].x - most));
    top = most;
  }
  float most = top;
#pragma unroll
  for (int o = 16; o > 0; o /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (top != neg_inf()) all *= tp_ex2(top - most);
#pragma unroll
  for (int o = 16; o > 0; o /= 2) all += __shfl_xor_sync(0xffffffffu, all, o);
  return make_float2(most, all);
}

// Blocks [0, joins): the segments of JOIN_WARPS / TEAM query heads joined, each by TEAM warps with
// the channels over the lanes, and the new token's rows stored.  Then blocks of MASS_SLOTS slots
// of a key head, which add the weights to `mass`.
constexpr int JOIN_WARPS = 8;

// KD: channels of a lane.
template <typename T, int TEAM, int KD>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_join_kernel(const PagedAttentionArgs a, int joins) {
  constexpr int THREADS = JOIN_WARPS * 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t G = a.block_heads, stride = (int64_t)a.c.heads * a.head_blocks * G;
  if ((int)blockIdx.x < joins) {
    __shared__ float sums[TEAM > 1 ? JOIN_WARPS : 1][32 * KD];
    const int row = blockIdx.x * (JOIN_WARPS / TEAM) + warp / TEAM, member = warp % TEAM;
    const bool there = row < a.B * a.H;
    const int b = there ? row / a.H : 0, h = there ? row - b * a.H : 0;
    const int kvh = h / a.group, in_group = h - kvh * a.group, D = a.c.channels;
    const int given = __ldg(a.lengths + b), n = there ? slots_of(a, b) : 0;
    T* const out = (T*)a.out + (int64_t)row * D;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float sum[KD] = {};
    float all = 1.0f;
    if (n > 0) {
      const int hblk = in_group / (int)G, g = in_group - hblk * (int)G;
      const int2 runs = a.runs_of[b];
      const int64_t first = segment(a, b, runs.x, kvh * a.head_blocks + hblk) * G + g;
      const float2* ml = a.ml + first;
      const float2 whole = whole_row(ml, stride, runs.y);
      all = whole.y;
      constexpr int AT_ONCE = 32 / KD;  // segments whose loads are under way together
      for (int s0 = member; s0 < runs.y; s0 += AT_ONCE * TEAM) {
        float f[AT_ONCE], x[AT_ONCE][KD];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          const int s = min(s0 + u * TEAM, runs.y - 1);
          f[u] = ml[s * stride].x;
          const float* p = a.part + (first + s * stride) * D;
#pragma unroll
          for (int k = 0; k < KD; ++k) x[u][k] = lane + 32 * k < D ? p[lane + 32 * k] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          const bool in = s0 + u * TEAM < runs.y;        // (an infinity twice, once times 0, would be NaN)
          f[u] = f[u] != neg_inf() ? tp_ex2(f[u] - whole.x) : 0.0f;
#pragma unroll
          for (int k = 0; k < KD; ++k) sum[k] += in ? x[u][k] * f[u] : 0.0f;
        }
      }
    }
    if constexpr (TEAM > 1) {
#pragma unroll
      for (int k = 0; k < KD; ++k) sums[warp][lane + 32 * k] = sum[k];
      __syncthreads();
      if (member > 0) return;
#pragma unroll
      for (int k = 0; k < KD; ++k)
#pragma unroll
        for (int w = 1; w < TEAM; ++w) sum[k] += sums[warp + w][lane + 32 * k];
    }
    if (!there) return;
    if (n == 0 && given != 0) {
      if (lane == 0) tp_record_index_error(a.bad.error, a.bad.seen);
      all = quiet_nan();
    }
#pragma unroll
    for (int k = 0; k < KD; ++k)
      if (lane + 32 * k < D) store_as(out + lane + 32 * k, sum[k] / all);
    if (a.key != nullptr && in_group == 0 && n > 0) {     // the new token's row to slot n - 1
      const int column = a.c.column(n - 1), in = a.c.within(n - 1, column);
      const int at = __ldg(a.c.table + (int64_t)b * a.c.table_row + column);
      if (at < 0 || at >= a.c.pages) return;
      const T* kn = (const T*)a.key + (int64_t)b * a.key_sb + (int64_t)kvh * a.key_sh;
      const T* vn = (const T*)a.value + (int64_t)b * a.value_sb + (int64_t)kvh * a.value_sh;
      T* kd = (T*)(a.c.k + (int64_t)at * a.c.k_page + (int64_t)in * a.c.k_slot + (int64_t)kvh * a.c.k_head);
      T* vd = (T*)(a.c.v + (int64_t)at * a.c.v_page + (int64_t)in * a.c.v_slot + (int64_t)kvh * a.c.v_head);
      for (int d = lane; d < D; d += 32) {
        kd[d] = kn[d];
        vd[d] = vn[d];
      }
    }
    return;
  }
  __shared__ float2 stat[64];
  const int chunks = (a.capacity + MASS_SLOTS - 1) / MASS_SLOTS;
  const int i = blockIdx.x - joins, chunk = i % chunks, kvh = i / chunks % a.c.heads,
            b = i / chunks / a.c.heads;
  const int n = slots_of(a, b);
  if (chunk * MASS_SLOTS >= n) return;
  constexpr int PER = MASS_SLOTS / THREADS;
  float* const mass = a.mass + (int64_t)b * a.mass_sb + (int64_t)kvh * a.mass_sh;
  const int slot0 = chunk * MASS_SLOTS + tid;
  float old[PER], sum[PER] = {};
#pragma unroll
  for (int k = 0; k < PER; ++k) {       // (a new token's slot begins)
    const int slot = slot0 + k * THREADS;
    old[k] = slot < n && !(a.key != nullptr && slot == n - 1) ? mass[slot] : 0.0f;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t head = (int64_t)b * a.H + (int64_t)kvh * a.group;
  const int2 runs = a.runs_of[b];
  for (int g0 = 0; g0 < a.group; g0 += 64) {
    const int some = min(64, a.group - g0);
    if (g0 > 0) __syncthreads();
    for (int g = warp; g < some; g += JOIN_WARPS) {
      const int hblk = (g0 + g) / (int)G, in = (g0 + g) - hblk * (int)G;
      const float2 row =
          whole_row(a.ml + segment(a, b, runs.x, kvh * a.head_blocks + hblk) * G + in, stride, runs.y);
      if (lane == 0) stat[g] = make_float2(row.x, 1.0f / row.y);
    }
    const float* sc = a.scores + (head + g0) * a.score_row + slot0;
    float x[PER];                       // (the first head's while the others find the sums)
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = slot0 + k * THREADS < n ? sc[k * THREADS] : neg_inf();
    __syncthreads();
    for (int g = 0; g < some; ++g) {
      const float2 st = stat[g];
      sc += a.score_row;
      float next[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) next[k] = g + 1 < some && slot0 + k * THREADS < n ? sc[k * THREADS] : neg_inf();
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        sum[k] += tp_ex2(x[k] - st.x) * st.y;
        x[k] = next[k];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int slot = slot0 + k * THREADS;
    if (slot < n) mass[slot] = old[k] + sum[k];
  }
}

// ---------------------------------------------------------------- launches
// Both kernels, the first with `smem` bytes of shared memory a block for tiles of `tile` slots.
template <typename T, typename K>
int attend_and_join(PagedAttentionArgs& a, K* kernel, size_t smem, int tile, int heads,
                    cudaStream_t stream) {
  int per_sm = 1;
  int st = resident_blocks((const void*)kernel, ATT_WARPS * 32, smem, per_sm);
  if (st != TP_OK) return st;
  a.block_heads = heads;
  a.head_blocks = (a.group + heads - 1) / heads;
  a.tile = tile;
  // as many runs as the SMs hold warps for by registers and shared memory (by the latter alone, 32 x 2048
  // gated slots of 4 query heads a key head ran as a wave and a half: 65 us for 54), with at least two
  // tiles each (four: 4 x 512 slots of 8 heads of 64 fp32 12.1 us for 10.0)
  per_sm = std::min(per_sm, ATT_MOST_BLOCKS);
  const int64_t subs = (int64_t)a.c.heads * a.head_blocks, tiles = a.B * ceil_div(a.capacity, tile);
  a.runs = (int)std::max<int64_t>(1, std::min((int64_t)num_sms() * per_sm * ATT_WARPS / subs, ceil_div(tiles, 2)));
  const int64_t blocks = ceil_div(a.runs * subs, ATT_WARPS);
  kernel<<<(unsigned)blocks, ATT_WARPS * 32, smem, stream>>>(a);
  st = launch_status();
  if (st != TP_OK) return st;
  // a warp joins the few segments of a head among many sequences, eight the many of one (48
  // sequences, 4 segments: 192 us with one warp, 203 with eight; one sequence, 148: 120 and 110)
  const int team = a.runs / a.B >= 8 ? JOIN_WARPS : 1;
  const int64_t joins = ceil_div((int64_t)a.B * a.H, JOIN_WARPS / team);
  int64_t joining = joins;
  if (a.mass) joining += (int64_t)a.B * a.c.heads * ceil_div(a.capacity, MASS_SLOTS);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)joining);
  cfg.blockDim = dim3(JOIN_WARPS * 32);
  cfg.stream = stream;
  // its blocks may be placed while the first kernel's last ones run; they wait for its end
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  auto run = [&](auto* one, auto* many) { return cuda_status(cudaLaunchKernelEx(&cfg, team > 1 ? many : one, a, (int)joins)); };
  return a.c.channels <= 64    ? run(paged_join_kernel<T, 1, 2>, paged_join_kernel<T, JOIN_WARPS, 2>)
         : a.c.channels <= 128 ? run(paged_join_kernel<T, 1, 4>, paged_join_kernel<T, JOIN_WARPS, 4>)
                               : run(paged_join_kernel<T, 1, 8>, paged_join_kernel<T, JOIN_WARPS, 8>);
}

template <typename T, int LPK, int NCH, int G, bool GATED, bool VEC>
int attend(PagedAttentionArgs& a, cudaStream_t stream) {
  // (two stages and twelve warps on an SM; three and eight: 32 x 2048 gated slots 31.5 us for 29.0)
  constexpr int STAGES = 2;
  return attend_and_join<T>(a, paged_attend_kernel<T, LPK, NCH, G, GATED, VEC, STAGES>,
                            (size_t)ATT_WARPS * STAGES * 2 * ATT_STEPS * NCH * 512,
                            ATT_STEPS * 32 / LPK, G, stream);
}

}  // namespace

}  // namespace tp
