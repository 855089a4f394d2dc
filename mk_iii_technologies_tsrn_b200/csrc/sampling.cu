// sampling.cu -- the next token of a language model from its logits and one given random
// number per row:
//
//   w_i = exp((x_i - max x) / temperature)
//   in the order of falling x (the lower index first of equals), keep the tokens that
//   are among the first top_k, have less than top_p of those' weight before them, and
//   weigh at least min_p (the best token always)
//   token = the first kept one, by index, where the running sum passes uniform * total
//
// A token is a whole number: a sum that is rounded one way here and another way there
// gives another token, so the weights are computed in 64 bits and summed as integers,
// w * 2^44 rounded: sums that no order changes, exact but for half a unit per token (a
// token below 2^-45 of the best is never taken).
//
// A row is a cluster of 1 to 8 blocks that exchange through shared memory.  Its logits are read
// once from DRAM and then from the L2.
//   - Without top_k and top_p: the maximum, the sum, and the part of the row where it is passed.
//   - With top_k: tokens are counted into bins of equal width below the maximum (of the threads'
//     best tokens alone, where top_k is far below the threads: a bin that holds top_k of those holds
//     as many tokens).  With top_p alone: the weights are added into the bins, exactly.
//   - The tokens of the bins up to the border go to one block, which sorts them, cuts them off
//     and finds the token.  Where they are more than CANDIDATES, those of the border's bin alone:
//     then the row has a threshold, and is read twice more as without filters.
//   - Where even that bin holds too many (flat rows, ties), and for a share of a top_k above
//     CANDIDATES, the threshold is found bit by bit over all tokens.
//
// Measured (in a CUDA graph): 16 x 256 fp32 without filters 5.4 us, 64 x 131072 bf16 with top_k
// around 50 and top_p 26 (2.6 us of bytes), 32 x 49999 fp32 with top_p 0.95 and 2300 tokens kept
// 37 to 39.  What bounds it is latency: passes of a few steps with an exchange of the cluster between
// them; in the last case half of it are instructions (weights in 64 bits).  Without filters 17 us at
// 32 x 49999 and 46 at 64 x 131072 bf16 (a weight for every token, twice), the best token alone 6 and 7.
// The search bit by bit takes up to 33 passes: 32 x 49999 equal logits 123 us with top_k, 147 with
// top_p, top_k of 5000 with top_p 184.
// 64 registers for 1024 threads: the bf16 form spills (188 bytes of stores, 248 of loads).
#include <algorithm>

#include "cluster.cuh"
#include "decode.cuh"

namespace tp {

namespace {

constexpr int BINS = 2048;
constexpr double UNIT = 17592186044416.0;       // 2^44
constexpr float REACH = 31.5f;                  // w < 2^-45 beyond this many units of temperature

template <int THREADS>
struct Shared {
  static constexpr int WARPS = THREADS / 32, CANDIDATES = THREADS;      // a candidate for each thread
  u64 exchange[2][2][MAX_CLUSTER];
  u64 reduce[2][WARPS];
  u64 candidate[2][CANDIDATES];        // of the bins before the border's, and of that
  u64 weight[CANDIDATES];
  u64 warp_sum[WARPS];
  u64 before_border, sum_all;
  double table[32];
  uint32_t low[BINS], high[BINS];      // counts, or weights in two halves
  int warp_ties[WARPS];
  int count[2], border;
  uint32_t cut;
  int ties;
};

// floats in order as unsigned numbers; NaN counts as -inf
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) x = -__int_as_float(0x7f800000);
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Add {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return a > b ? a : b; }
};

__device__ __forceinline__ u64 warp_inclusive(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// Sum of sums[0 .. warp) over a block's warps, and of all of them.
template <int WARPS>
__device__ __forceinline__ u64 before_warp(const u64* sums, int warp, int lane, u64& all) {
  const u64 mine = lane < WARPS ? sums[lane] : 0, upto = warp_inclusive(mine, lane);
  all = __shfl_sync(0xffffffffu, upto, WARPS - 1);
  return __shfl_sync(0xffffffffu, upto - mine, warp);
}

// A warp's part of a row, in steps of 16 bytes a lane.  They lie on 16-byte boundaries wherever the
// row begins; where a step reaches over an end of the row it takes single numbers, and -inf for those
// that are not there.
template <typename T>
struct Row {
  static constexpr int PER = 16 / sizeof(T);      // tokens of a lane's step, next to one another
  const T* x;
  int off, begin, end;                            // tokens before x to a boundary; part, counted from there

  __device__ __forceinline__ Row(const T* row, int V, int part, int parts) : x(row) {
    off = (int)(((uintptr_t)row & 15) / sizeof(T));
    const int per = ((V + off + parts - 1) / parts + PER - 1) / PER * PER;
    const int64_t first = (int64_t)part * per;
    begin = (int)min((int64_t)V + off, first);
    end = (int)min((int64_t)V + off, first + per);
  }
  // f(index of the first, values) of each step of this lane; the whole warp runs every step.  AHEAD:
  // the next step's numbers are asked for before this one's are looked at (where that leaves
  // registers for it).
  template <bool AHEAD = false, typename F>
  __device__ __forceinline__ void each(F f) const {
    const int lane_at = ((int)threadIdx.x & 31) * PER;
    auto whole = [&](int p) { return p >= off && p + PER <= end; };
    auto get = [&](int p) { return __ldg((const uint4*)(x + (p - off))); };
    uint4 next = make_uint4(0, 0, 0, 0);
    if (AHEAD && whole(begin + lane_at)) next = get(begin + lane_at);
    for (int p0 = begin; p0 < end; p0 += 32 * PER) {
      const int p = p0 + lane_at;
      uint4 u = next;
      if (AHEAD && whole(p + 32 * PER)) next = get(p + 32 * PER);
      float v[PER];
      if (whole(p)) {
        if (!AHEAD) u = get(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[2 * k] = __uint_as_float(w[k] << 16);
            v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k)
          v[k] = p + k >= off && p + k < end ? tp_load_as_f32<T>(x + (p + k - off))
                                             : -__int_as_float(0x7f800000);
      }
      f(p - off, v);
    }
  }
};

// w = exp((x - top) / temperature) = 2^t as 2^n 2^(j / 32) 2^f with |f| <= 1 / 64: the middle factor
// from a table, the last by its Taylor series to f^5 (the rest is below (ln 2 / 64)^6 / 720 <
// 2^-48).  An exponential of full precision and its conversion to an integer took 100 instructions
// of a token, this takes 25.
struct Weights {
  float top;
  double top64, per, per2;        // the maximum, 1 / temperature, and that for base 2
  const double* table;            // 2^(j / 32)
  __device__ __forceinline__ double real(float x) const {
    const double t = ((double)x - top64) * per2;
    const double shift = 0x1.8p47;                       // t to a 32nd, in its low bits
    const double s = t + shift, f = t - (s - shift);
    const int at = __double2loint(s), j = at & 31, n = at >> 5;
    const double z = f * 0.693147180559945309417;
    double p = fma(z, 1.0 / 120, 1.0 / 24);
    p = fma(z, p, 1.0 / 6);
    p = fma(z, p, 0.5);
    p = fma(z, p, 1.0);
    p = fma(z, p, 1.0) * table[j];
    const double w = __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
    return x == top ? 1.0 : t > -60.0 ? w : 0.0;         // (of NaN nothing)
  }
  // w * 2^44 to the nearest, read from the low bits of a sum
  __device__ __forceinline__ u64 whole(double w) const {
    return (u64)__double_as_longlong(fma(w, UNIT, 0x1p52)) & 0xfffffffffffffull;
  }
};

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) sample_kernel(const SampleArgs a, int cluster) {
  constexpr int WARPS = THREADS / 32, CANDIDATES = THREADS;
  __shared__ Shared<THREADS> s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank();
  const int64_t b = blockIdx.x / cluster;
  const int V = (int)a.V;
  if (cluster > 1) cluster_arrive();

  const Row<T> row((const T*)a.logits + b * a.ld, V, (int)rank * WARPS + warp, cluster * WARPS);

  // (asked for before the logits: their loads are under way together)
  const double temperature = a.temperature.of_row ? (double)a.temperature.of_row[b] : a.temperature.all;
  const double top_p = a.top_p.of_row ? (double)a.top_p.of_row[b] : a.top_p.all;
  const double min_p = a.min_p.of_row ? (double)a.min_p.of_row[b] : a.min_p.all;
  const int64_t asked = a.top_k_of_row ? (int64_t)a.top_k_of_row[b] : a.top_k;
  const double u = a.uniform64 ? ((const double*)a.uniform)[b] : (double)((const float*)a.uniform)[b];
  const bool by_k = asked > 0 && asked < V, by_p = top_p < 1.0;
  const int top_k = by_k ? (int)asked : V;

  // Sum (or maximum) of v over the cluster's threads.  Two calls' slots never meet: a block is
  // past a call's barrier only when all have read the one before.
  int calls = 0;
  auto meet = [&] {
    if (cluster > 1) cluster_sync();
    else __syncthreads();
  };
  auto all = [&](u64 v, int which, auto op) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) s.reduce[which][warp] = v;
  };
  auto finish = [&](int which, auto op) {         // after a __syncthreads: one warp, to every block
    u64 v = lane < WARPS ? s.reduce[which][lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane < cluster) remote_store(remote(&s.exchange[calls & 1][which][rank], lane), v);
  };
  auto joined = [&](int which, auto op) {
    u64 v = 0;
    for (int r = 0; r < cluster; ++r) v = op(v, s.exchange[calls & 1][which][r]);
    return v;
  };
  auto reduce = [&](u64 v, auto op) {
    all(v, 0, op);
    __syncthreads();
    if (warp == 0) finish(0, op);
    meet();
    const u64 r = joined(0, op);
    ++calls;
    return r;
  };

  // ---- the best token, of this thread and of all; the lowest number
  if (tid < 2) s.count[tid] = 0;
  if (tid < 32) s.table[tid] = exp2(tid / 32.0);
  for (int i = tid; i < BINS; i += THREADS) s.low[i] = s.high[i] = 0;
  const float inf = __int_as_float(0x7f800000);
  float mine_best = -inf, lowest = inf;
  int mine_at = 0;                      // (a row without a token above -inf is none to take from)
  const bool of_threads = by_k && top_k <= cluster * THREADS / 8 && V >= cluster * THREADS;
  row.template each<true>([&](int i, const float* v) {
    float top = v[0];
#pragma unroll
    for (int k = 1; k < Row<T>::PER; ++k) top = fmaxf(top, v[k]);      // (NaN is not)
    if (top > mine_best) {              // the first of equals
      mine_best = top;
#pragma unroll
      for (int k = Row<T>::PER - 1; k >= 0; --k) mine_at = v[k] == top ? i + k : mine_at;
    }
    if ((by_k || by_p) && !of_threads) {
#pragma unroll
      for (int k = 0; k < Row<T>::PER; ++k) lowest = fminf(lowest, v[k] > -inf ? v[k] : inf);
    }
  });
  u64 best = (u64)key_of(mine_best) << 32 | (0xffffffffu - (uint32_t)mine_at);
  uint32_t least = ~key_of(lowest);     // (the largest of the inverted keys)
  all(best, 0, Max());
  all(least, 1, Max());
  __syncthreads();
  if (cluster > 1) cluster_wait();      // every block of the row runs
  if (warp == 0) {
    finish(0, Max());
    finish(1, Max());
  }
  meet();
  best = joined(0, Max());
  least = (uint32_t)joined(1, Max());
  ++calls;
  Weights wt;
  wt.top = value_of((uint32_t)(best >> 32));
  const int first = (int)(0xffffffffu - (uint32_t)best);
  const bool leader = rank == 0 && tid == 0;
  if (wt.top == -inf) {                   // nothing to take
    if (leader) {
      a.token[b] = -1;
      if (a.logprob) a.logprob[b] = __int_as_float(0x7fc00000);
    }
    return;
  }
  if (!(temperature > 0.0) || top_k == 1 || top_p <= 0.0 || min_p > 1.0) {
    if (leader) {
      a.token[b] = first;
      if (a.logprob) a.logprob[b] = 0.0f;
    }
    return;
  }
  wt.top64 = (double)wt.top;
  wt.per = 1.0 / temperature;
  wt.per2 = wt.per * 1.44269504088896340736;
  wt.table = s.table;
  // the place in the running sum: the first token whose sum is above it
  auto place = [&](u64 total) {
    const double t = u * (double)total;
    return t >= 0.0 && t < (double)total ? min((u64)t, total - 1) : (t < 0.0 ? 0ull : total - 1);
  };
  auto write = [&](int token, float x, u64 total) {
    a.token[b] = token;
    if (a.logprob)
      a.logprob[b] = (float)((x == wt.top ? 0.0 : ((double)x - wt.top64) * wt.per) - log((double)total / UNIT));
  };

  uint32_t cut = 0;                     // kept: keys above it, and the first `ties` equal to it
  int64_t ties = INT64_MAX;
  if (by_k || by_p) {
    // ---- bins below the maximum, down to the lowest number or to where a token weighs nothing
    const float span = of_threads ? inf : wt.top - value_of(~least);
    const float reach = fminf(fminf((float)(REACH * temperature), span), 3e38f), bins_per = BINS / reach;
    auto bin_of = [&](float x) {        // BINS: weighs nothing
      if (x == wt.top) return 0;
      const float d = wt.top - x;
      return d <= reach ? min(BINS - 1, (int)(d * bins_per)) : BINS;
    };
    if (of_threads) {
      const int bin = bin_of(mine_best);
      if (bin < BINS) atomicAdd(&s.low[bin], 1u);
    } else {
      row.each([&](int i, const float* v) {
#pragma unroll
        for (int k = 0; k < Row<T>::PER; ++k) {
          const int bin = bin_of(v[k]);
          if (bin >= BINS) continue;
          if (by_k) {
            atomicAdd(&s.low[bin], 1u);
          } else {
            const u64 w = wt.whole(wt.real(v[k]));
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.low[bin], lo);
            const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old);
            if (hi) atomicAdd(&s.high[bin], hi);
          }
        }
      });
    }
    meet();
    if (rank == 0) {                    // the border's bin: the first where the sum reaches it
      constexpr int EACH = BINS / THREADS;
      u64 mine[EACH], at = 0;
#pragma unroll
      for (int k = 0; k < EACH; ++k) mine[k] = 0;
#pragma unroll
      for (int r = 0; r < MAX_CLUSTER; ++r) {          // (without a turn's loads waiting for the last's)
        if (r >= cluster) continue;
        uint32_t low[EACH], high[EACH];
#pragma unroll
        for (int k = 0; k < EACH; ++k) low[k] = remote_load(remote(&s.low[EACH * tid + k], r));
#pragma unroll
        for (int k = 0; k < EACH; ++k) high[k] = by_k ? 0 : remote_load(remote(&s.high[EACH * tid + k], r));
#pragma unroll
        for (int k = 0; k < EACH; ++k) mine[k] += (u64)high[k] << 32 | low[k];
      }
#pragma unroll
      for (int k = 0; k < EACH; ++k) at += mine[k];
      const u64 own = at;
      at = warp_inclusive(at, lane);
      if (lane == 31) s.warp_sum[warp] = at;
      if (tid == 0) s.border = BINS;
      __syncthreads();
      u64 everything;
      at += before_warp<WARPS>(s.warp_sum, warp, lane, everything) - own;
      // (with top_k above the universe's tokens: the last bin that has any)
      auto reaches = [&](u64 sum) {
        return by_k ? sum >= min((u64)top_k, everything) : (double)sum >= top_p * (double)everything;
      };
      if (!reaches(at) && reaches(at + own) && !(of_threads && everything < (u64)top_k)) {
        bool found = false;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
          if (!found && reaches(at + mine[k])) {
            found = true;
            s.border = EACH * tid + k;
            s.before_border = at;
            s.sum_all = everything;
          }
          at += mine[k];
        }
      }
      // (fewer threads with a token than top_k: all tokens that weigh something)
      if (of_threads && everything < (u64)top_k && tid == 0) s.border = BINS - 1;
      __syncthreads();
      if (tid > 0 && tid < cluster) {
        remote_store(remote(&s.border, tid), s.border);
        remote_store(remote(&s.sum_all, tid), s.sum_all);
      }
    }
    meet();
    const int border = s.border;
    // ---- gather: the border's bin and, at once under top_k, where they are needed as a rule, the
    // bins before it; under top_p these are counted first
    // (no token below `floor` is in them: the border's far end with more than its rounding to spare)
    const float floor = border < BINS - 1 ? wt.top - (border + 2) / bins_per : -inf;
    auto gather = [&](bool before, bool at_border) {
      int counted = 0;
      row.template each<true>([&](int i, const float* v) {
        bool any = false;
#pragma unroll
        for (int k = 0; k < Row<T>::PER; ++k) any |= v[k] >= floor;
        if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
        for (int k = 0; k < Row<T>::PER; ++k) {
          const int bin = bin_of(v[k]);
          counted += bin < border;
#pragma unroll
          for (int list = 0; list < 2; ++list) {
            const bool take = list ? at_border && bin == border && bin < BINS : before && bin < border;
            const uint32_t takers = __ballot_sync(0xffffffffu, take);
            if (!takers) continue;
            int at = 0;
            if (lane == __ffs(takers) - 1) at = remote_add(remote(&s.count[list], 0), __popc(takers));
            at = __shfl_sync(0xffffffffu, at, __ffs(takers) - 1) + __popc(takers & ((1u << lane) - 1));
            if (take && at < CANDIDATES)
              remote_store(remote(&s.candidate[list][at], 0),
                           (u64)key_of(v[k]) << 32 | (0xffffffffu - (uint32_t)(i + k)));
          }
        }
      });
      return counted;
    };
    if (by_k) {
      gather(true, true);
    } else {
      const u64 counted = reduce((u64)gather(false, true), Add());
      // (the border's tokens are in rank 0's count, which only it may look at before a barrier)
      if (counted <= CANDIDATES) gather(true, false);
      else if (rank == 0 && tid == 0) s.count[0] = (int)counted;
    }
    meet();
    if (rank == 0 && tid > 0 && tid < cluster) {
      remote_store(remote(&s.count[0], tid), s.count[0]);
      remote_store(remote(&s.count[1], tid), s.count[1]);
    }
    meet();
    const int above = s.count[0], in_border = s.count[1], count = above + in_border;
    const u64 sum_all = s.sum_all;      // (under top_p alone: the weight of all)
    const bool few = count <= CANDIDATES;
    const bool one_bin = !few && in_border <= CANDIDATES && !(of_threads && above >= top_k);
    if (few && rank != 0) return;
    if (few || one_bin) {
      // ---- sort, cut off, sort by index, find the place (or, of one bin, the threshold)
      auto sort = [&](u64 v, int n) {   // falling; threads from n on hold zeros
        for (int k = 2; k <= n; k *= 2)
          for (int j = k / 2; j > 0; j /= 2) {
            u64 other;
            if (j >= 32) {
              s.candidate[0][tid] = v;
              __syncthreads();
              other = s.candidate[0][tid ^ j];
              __syncthreads();
            } else if (tid < n) {       // (whole warps)
              other = __shfl_xor_sync(0xffffffffu, v, j);
            } else {
              continue;
            }
            const bool larger = ((tid & j) == 0) == ((tid & k) == 0);
            v = (v > other) == larger ? v : other;
          }
        return v;
      };
      auto scan = [&](u64 w) {          // inclusive over the block
        u64 at = warp_inclusive(w, lane);
        if (lane == 31) s.warp_sum[warp] = at;
        __syncthreads();
        u64 sum;
        at += before_warp<WARPS>(s.warp_sum, warp, lane, sum);
        __syncthreads();
        return at;
      };
      if (rank == 0) {
        const int listed = few ? count : in_border, skipped = few ? 0 : above;
        int size = 32;
        while (size < listed) size *= 2;
        u64 v = 0;
        if (tid < listed) v = few && tid < above ? s.candidate[0][tid] : s.candidate[1][few ? tid - above : tid];
        __syncthreads();
        v = sort(v, size);
        const bool there = tid < listed && skipped + tid < top_k;
        const float x = value_of((uint32_t)(v >> 32));
        const double w = there ? wt.real(x) : 0.0;
        const u64 whole = wt.whole(w);
        const u64 sum = scan(whole) + (one_bin && !by_k ? s.before_border : 0);
        if (tid == THREADS - 1) s.weight[0] = sum;
        __syncthreads();
        const u64 share = by_k ? s.weight[0] : sum_all;
        bool keep = there;
        if (by_p && !(one_bin && by_k)) keep = keep && (double)(sum - whole) < top_p * (double)share;
        if (one_bin) {                  // the last one kept, and how many equal to it are
          const int n = __syncthreads_count(keep);
          s.candidate[0][tid] = v;
          __syncthreads();
          const uint32_t last = (uint32_t)(s.candidate[0][max(n - 1, 0)] >> 32);
          const bool same = tid < listed && (uint32_t)(v >> 32) == last;
          const int equal = __syncthreads_count(keep && same), all_equal = __syncthreads_count(same);
          if (tid < cluster) {
            remote_store(remote(&s.cut, tid), (int)last);
            remote_store(remote(&s.ties, tid), equal == all_equal ? -1 : equal);      // -1: all
          }
        } else {
          keep = (keep && w >= min_p) || tid == 0;
          __syncthreads();
          s.weight[tid] = whole;
          const uint32_t index = 0xffffffffu - (uint32_t)v;
          // falling again: the lowest index first; what is not kept last
          u64 o = keep ? (u64)(0xffffffffu - index) << 32 | (uint32_t)(tid + 1) : 0;
          o = sort(o, size);
          __syncthreads();
          const int from = (int)(uint32_t)o - 1;
          const u64 ow = from >= 0 ? s.weight[from] : 0;
          const u64 run = scan(ow);
          s.candidate[0][tid] = v;      // (by rank)
          if (tid == THREADS - 1) s.reduce[0][0] = run;
          __syncthreads();
          const u64 total = s.reduce[0][0], t = place(total);
          if (ow > 0 && run > t && run - ow <= t)
            write((int)(0xffffffffu - (uint32_t)(o >> 32)),
                  value_of((uint32_t)(s.candidate[0][from] >> 32)), total);
          return;
        }
      }
      meet();
      cut = s.cut;
      ties = s.ties < 0 ? INT64_MAX : s.ties;
    }
    // ---- bit by bit over all tokens
    auto weigh_from = [&](uint32_t key) {
      u64 sum = 0;
      row.each([&](int i, const float* v) {
#pragma unroll
        for (int k = 0; k < Row<T>::PER; ++k)
          if (key_of(v[k]) >= key) sum += wt.whole(wt.real(v[k]));
      });
      return reduce(sum, Add());
    };
    auto count_from = [&](uint32_t key) {
      u64 sum = 0;
      row.each([&](int i, const float* v) {
#pragma unroll
        for (int k = 0; k < Row<T>::PER; ++k) sum += key_of(v[k]) >= key;
      });
      return reduce(sum, Add());
    };
    // (no key of a token is 2^32 - 1, so that cut + 1 is one)
    u64 share = sum_all;
    if (by_k) {
      if (!one_bin) {
        for (uint32_t bit = 1u << 31; bit; bit >>= 1)
          if (count_from(cut | bit) >= (u64)top_k) cut |= bit;
        ties = top_k - (int64_t)count_from(cut + 1);
      }
      if (by_p)
        share = ties == INT64_MAX ? weigh_from(cut)
                                  : weigh_from(cut + 1) + (u64)ties * wt.whole(wt.real(value_of(cut)));
    }
    if (by_p && !(one_bin && !by_k)) {
      const double wanted = top_p * (double)share;
      uint32_t p = 0;
      for (uint32_t bit = 1u << 31; bit; bit >>= 1)
        if ((double)weigh_from(p | bit) >= wanted) p |= bit;
      if (p >= cut) {
        const u64 above_p = weigh_from(p + 1), one = wt.whole(wt.real(value_of(p)));
        // the first of the ties whose sum before it reaches the share is left out
        int64_t r = one > 0 ? (int64_t)ceil((wanted - (double)above_p) / (double)one) : INT64_MAX;
        r = max(r, (int64_t)1);
        ties = p > cut ? r : min(ties, r);
        cut = p;
      }
    }
  }

  // ---- the place among the kept tokens, by index
  int64_t tie_base = 0;
  if (ties != INT64_MAX) {
    u64 mine = 0;
    row.each([&](int i, const float* v) {
#pragma unroll
      for (int k = 0; k < Row<T>::PER; ++k) mine += key_of(v[k]) == cut;
    });
#pragma unroll
    for (int o = 16; o > 0; o /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __syncthreads();
    if (lane == 0) s.warp_ties[warp] = (int)mine;
    (void)reduce(lane == 0 ? mine : 0, Add());
    for (int w = 0; w < warp; ++w) tie_base += s.warp_ties[w];
    for (uint32_t r = 0; r < rank; ++r) tie_base += (int64_t)s.exchange[(calls - 1) & 1][0][r];
  }
  // weights of a step's tokens; `base`: ties before the step
  auto kept = [&](int i, const float* v, int64_t& base, u64 (&w)[Row<T>::PER]) {
    int mine = 0;
#pragma unroll
    for (int k = 0; k < Row<T>::PER; ++k) mine += key_of(v[k]) == cut;
    int64_t at = base;
    if (ties != INT64_MAX) {
      const int upto = (int)warp_inclusive(mine, lane);
      at += upto - mine;
      base += __shfl_sync(0xffffffffu, upto, 31);
    }
    bool in[Row<T>::PER], any = false;
#pragma unroll
    for (int k = 0; k < Row<T>::PER; ++k) {
      const uint32_t key = key_of(v[k]);
      const bool tie = key == cut;
      in[k] = key > cut || (tie && at < ties);
      any |= in[k];
      at += tie;
      w[k] = 0;
    }
    if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
    for (int k = 0; k < Row<T>::PER; ++k) {            // (all of them, rather than one after another)
      const double real = wt.real(v[k]);
      if (in[k] && (real >= min_p || i + k == first)) w[k] = wt.whole(real);
    }
  };
  u64 sum = 0;
  {
    int64_t base = tie_base;
    row.each([&](int i, const float* v) {
      u64 w[Row<T>::PER];
      kept(i, v, base, w);
#pragma unroll
      for (int k = 0; k < Row<T>::PER; ++k) sum += w[k];
    });
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) s.warp_sum[warp] = sum;
  const u64 total = reduce(lane == 0 ? sum : 0, Add());
  u64 own_block;
  u64 before = before_warp<WARPS>(s.warp_sum, warp, lane, own_block);
  for (uint32_t r = 0; r < rank; ++r) before += s.exchange[(calls - 1) & 1][0][r];
  const u64 t = place(total);
  if (!(before <= t && t < before + sum)) return;                // another warp's
  int64_t base = tie_base;
  u64 run = before;
  row.each([&](int i, const float* v) {
    u64 w[Row<T>::PER], mine = 0;
    kept(i, v, base, w);
#pragma unroll
    for (int k = 0; k < Row<T>::PER; ++k) mine += w[k];
    const u64 upto = run + warp_inclusive(mine, lane);
    u64 at = upto - mine;
    if (at <= t && t < upto) {
#pragma unroll
      for (int k = 0; k < Row<T>::PER; ++k) {
        if (at <= t && t < at + w[k]) write(i + k, v[k], total);
        at += w[k];
      }
    }
    run = __shfl_sync(0xffffffffu, upto, 31);
  });
}

template <typename T, int THREADS>
int sample(const SampleArgs& a, cudaStream_t stream) {
  constexpr int WARPS = THREADS / 32;
  // as many blocks for a row as leave its warps a few steps, while the SMs hold all rows' at once
  // (32 x 49999: 69 us with one block, 38 with four, 81 with eight, which take turns; 64 x 131072:
  // 30, 26 with two, 72 with eight)
  int cluster = 1;
  while (cluster < MAX_CLUSTER && a.V > (int64_t)cluster * WARPS * 64 * (16 / (int)sizeof(T)) &&
         a.B * cluster * 2 <= num_sms())
    cluster *= 2;
  TP_RETURN_IF(a.B * cluster > INT32_MAX, TP_ERR_TOO_LARGE);
  return launch_clusters(sample_kernel<T, THREADS>, a.B * cluster, THREADS, cluster, stream, a, cluster);
}

}  // namespace

int launch_sample_tokens(const SampleArgs& a, cudaStream_t stream) {
  // (a small vocabulary in small blocks, whose barriers are shorter: 16 rows of 256 logits
  // 10.5 us in blocks of 1024, 7.5 in these at that stage, 5.5 now, the launch among them)
  const bool small = a.V <= 4096;
  if (a.dtype == TP_DTYPE_BF16)
    return small ? sample<uint16_t, 256>(a, stream) : sample<uint16_t, 1024>(a, stream);
  return small ? sample<float, 256>(a, stream) : sample<float, 1024>(a, stream);
}

}  // namespace tp
