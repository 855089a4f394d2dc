// paged_attention.cuh -- attention of one new token per sequence over a paged key-value
// cache (paged_attention_{f32,bf16}.cu instantiate it):
//
//   s_j = scale / tau * ((1 - g) q . k_j + g max_f(q_f + k_jf))      (without gate: q . k_j)
//   o   = sum_j softmax(s)_j v_j,  j < lengths[b]
//
// the decoding form of the blended score of the tropical attention modules
// (tropformer_dropin.py:236-260) with grouped query heads.
//
// Every byte of K and V is read once and used for `group` query heads: bound by DRAM.
// A warp takes tiles of TK slots.  A slot's channels lie over LPK lanes, 16 bytes each,
// so that a load instruction of the warp reads 32 / LPK whole rows; eight such steps
// make a tile (4 KB of K and 4 KB of V a chunk).  Rows come through asynchronous copies
// into shared memory, STAGES - 1 tiles ahead; every lane copies what it reads itself, so
// that no barrier is needed.  The eight partial sums of a lane are joined over the lanes
// by halves (4 + 2 + 1 shuffles for eight sums), which leaves each lane a slot's score.
// Softmax statistics run along (maximum and sum, base 2) in fp32; the sums over V stay in
// registers.  A row is cut into `splits` blocks over its length where there are few rows,
// joined by a second kernel that also adds the weights to `mass`.
#pragma once

#include "decode.cuh"

namespace tp {

namespace {

constexpr int ATT_WARPS = 4;
constexpr int ATT_STEPS = 8;

__device__ __forceinline__ float neg_inf() { return -__int_as_float(0x7f800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ int reversed3(int i) {
  return ((i & 1) << 2) | (i & 2) | ((i >> 2) & 1);
}

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

// T: float, or uint16_t for bf16.  LPK lanes of a slot with NCH chunks of 16 bytes each; G
// query heads at a time; VEC: every row begins and ends on 16 bytes.
template <typename T, int LPK, int NCH, int G, bool GATED, bool VEC, int STAGES>
struct PagedAttend {
  static constexpr int N = Chunk<T>::N;
  static constexpr int KPL = 32 / LPK;                       // slots of a load
  static constexpr int TK = ATT_STEPS * KPL;                 // slots of a tile
  static constexpr int STAGE = 2 * ATT_STEPS * NCH * 32;     // 16-byte pieces of a warp's stage
  static constexpr int DP = LPK * NCH * N;
  static constexpr size_t RING = (size_t)ATT_WARPS * STAGES * STAGE * 16;
  static constexpr size_t JOIN = (size_t)ATT_WARPS * G * (DP + 2) * 4 + 16;
  static constexpr size_t SMEM = RING > JOIN ? RING : JOIN;
};

template <typename T, int LPK, int NCH, int G, bool GATED, bool VEC, int STAGES>
__global__ void __launch_bounds__(ATT_WARPS * 32)
paged_attend_kernel(const PagedAttentionArgs a) {
  using P = PagedAttend<T, LPK, NCH, G, GATED, VEC, STAGES>;
  constexpr int N = P::N, N2 = N / 2, KPL = P::KPL, TK = P::TK;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / LPK, c = lane % LPK;
  const int split = blockIdx.x % a.splits;
  int r = blockIdx.x / a.splits;
  const int hblk = r % a.head_blocks;
  r /= a.head_blocks;
  const int kvh = r % a.c.heads, b = r / a.c.heads;
  const int D = a.c.channels;

  int n = __ldg(a.lengths + b);
  bool bad = n < 0 || n > a.capacity;
  if (bad && threadIdx.x == 0) tp_record_index_error(a.bad.error, a.bad.seen);
  n = n < 0 ? 0 : min(n, a.capacity);
  const bool has_new = a.key != nullptr && !bad && n > 0;
  const int parts = paged_splits(n, a.splits, a.unit);
  if (split >= parts) return;
  const int tiles = (n + TK - 1) / TK;
  const int t0 = (int)((int64_t)split * tiles / parts), t1 = (int)((int64_t)(split + 1) * tiles / parts);

  // the query's channels of this lane
  float2 q[G][NCH][N2];
  float factor[G], blend[G];
  int h_of[G];
  int valid[NCH];              // channels of this lane's chunks
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) valid[ch] = max(0, min(N, D - (c + ch * LPK) * N));
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int in_group = hblk * G + g;
    const bool there = in_group < a.group;
    const int h = kvh * a.group + (there ? in_group : 0);
    h_of[g] = there ? h : -1;
    const T* src = (const T*)a.q + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      float e[N];
#pragma unroll
      for (int i = 0; i < N; ++i)
        e[i] = there && i < valid[ch] ? tp_load_as_f32<T>(src + (c + ch * LPK) * N + i) : 0.0f;
#pragma unroll
      for (int i = 0; i < N2; ++i) q[g][ch][i] = make_float2(e[2 * i], e[2 * i + 1]);
    }
    factor[g] = (a.tau ? a.scale / __ldg(a.tau + h) : a.scale) * 1.4426950408889634f;
    blend[g] = GATED ? __ldg(a.gate + (int64_t)b * a.H + h) : 0.0f;
  }

  const int* row = a.c.table + (int64_t)b * a.c.table_row;
  const char* const khead = a.c.k + (int64_t)kvh * a.c.k_head;
  const char* const vhead = a.c.v + (int64_t)kvh * a.c.v_head;
  const char* const knew = has_new ? (const char*)((const T*)a.key + (int64_t)b * a.key_sb + (int64_t)kvh * a.key_sh) : nullptr;
  const char* const vnew = has_new ? (const char*)((const T*)a.value + (int64_t)b * a.value_sb + (int64_t)kvh * a.value_sh) : nullptr;
  uint4* const ring = (uint4*)smem + (size_t)warp * STAGES * P::STAGE + lane;

  // this lane's slot of a tile: the page is asked for one tile before it is needed
  const int mine = t1 - t0 > warp ? (t1 - t0 - warp + ATT_WARPS - 1) / ATT_WARPS : 0;
  auto slot_of = [&](int i) { return (t0 + warp + i * ATT_WARPS) * TK + lane; };
  auto page_of = [&](int i) {
    const int s = slot_of(i);
    return i < mine && lane < TK && s < n ? __ldg(row + s / a.c.page_size) : 0;
  };
  int page = page_of(0);
  auto issue = [&](int i) {
    if (i < mine) {
      const int s = slot_of(i);
      const char *kp = nullptr, *vp = nullptr;
      if (lane < TK && s < n) {
        if (page < 0 || page >= a.c.pages) {
          tp_record_index_error(a.bad.error, a.bad.seen);
          bad = true;
        } else if (has_new && s == n - 1) {
          kp = knew;
          vp = vnew;
        } else {
          const int in = s % a.c.page_size;
          kp = khead + (int64_t)page * a.c.k_page + (int64_t)in * a.c.k_slot;
          vp = vhead + (int64_t)page * a.c.v_page + (int64_t)in * a.c.v_slot;
        }
      }
      page = page_of(i + 1);
      uint4* dst = ring + (size_t)(i % STAGES) * P::STAGE;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
        for (int step = 0; step < ATT_STEPS; ++step) {
          const char* p = shfl_ptr(kv ? vp : kp, step * KPL + sub);
#pragma unroll
          for (int ch = 0; ch < NCH; ++ch, dst += 32) {
            const int off = (c + ch * LPK) * 16;
            if constexpr (VEC) {
              const bool get = p != nullptr && valid[ch] > 0;
              tp_cp_async16(dst, get ? p + off : (const char*)a.lengths, get ? 16 : 0);
            } else {
              alignas(16) T e[N];
#pragma unroll
              for (int x = 0; x < N; ++x)
                e[x] = p != nullptr && x < valid[ch] ? *((const T*)(p + off) + x) : T(0);
              *dst = *(const uint4*)e;
            }
          }
        }
      }
    }
    tp_cp_async_commit();
  };

  float m[G], l[G];
  float2 acc[G][NCH][N2];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = neg_inf();
    l[g] = 0.0f;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int i = 0; i < N2; ++i) acc[g][ch][i] = make_float2(0.0f, 0.0f);
  }

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i);
  for (int i = 0; i < mine; ++i) {
    issue(i + STAGES - 1);
    tp_cp_async_wait<STAGES - 1>();
    const uint4* kst = ring + (size_t)(i % STAGES) * P::STAGE;
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

    const int key = (t0 + warp + i * ATT_WARPS) * TK + reversed3(c & 7) * KPL + sub;
    float p[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float s = join_steps<LPK>(dot[g], lane, [](float x, float y) { return x + y; });
      if constexpr (GATED) {
        const float t = join_steps<LPK>(trop[g], lane, [](float x, float y) { return tp_max_nan(x, y); });
        s = blend[g] * t + (1.0f - blend[g]) * s;
      }
      s = key < n ? s * factor[g] : neg_inf();
      if (a.scores != nullptr && c < 8 && key < n && h_of[g] >= 0)
        a.scores[((int64_t)b * a.H + h_of[g]) * a.capacity + key] = s;
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
  }
  tp_cp_async_wait<0>();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // lanes, then warps
#pragma unroll
  for (int g = 0; g < G; ++g) {
    l[g] = c < 8 ? l[g] : 0.0f;
#pragma unroll
    for (int o = 1; o < 32; o *= 2)
      if (o < 8 || o >= LPK) l[g] += __shfl_xor_sync(0xffffffffu, l[g], o);
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int x = 0; x < N2; ++x)
#pragma unroll
        for (int o = LPK; o < 32; o *= 2) {
          acc[g][ch][x].x += __shfl_xor_sync(0xffffffffu, acc[g][ch][x].x, o);
          acc[g][ch][x].y += __shfl_xor_sync(0xffffffffu, acc[g][ch][x].y, o);
        }
  }
  bad = __syncthreads_or(bad);              // (and every warp is done with the ring)
  float* const sums = (float*)smem;         // [warp][g][DP]
  float2* const stats = (float2*)(sums + ATT_WARPS * G * P::DP);
  if (sub == 0) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
        for (int x = 0; x < N2; ++x)
          *(float2*)(sums + (warp * G + g) * P::DP + (c + ch * LPK) * N + 2 * x) = acc[g][ch][x];
      if (c == 0) stats[warp * G + g] = make_float2(m[g], l[g]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * P::DP; i += ATT_WARPS * 32) {
    const int g = i / P::DP, d = i % P::DP;
    if (hblk * G + g >= a.group || d >= D) continue;
    const int h = kvh * a.group + hblk * G + g;
    float top = neg_inf();
#pragma unroll
    for (int w = 0; w < ATT_WARPS; ++w) top = fmaxf(top, stats[w * G + g].x);
    float sum = 0.0f, all = 0.0f;
#pragma unroll
    for (int w = 0; w < ATT_WARPS; ++w) {
      const float2 s = stats[w * G + g];
      const float f = s.x == neg_inf() ? 0.0f : tp_ex2(s.x - top);
      all += s.y * f;
      sum += sums[(w * G + g) * P::DP + d] * f;
    }
    if (bad) all = quiet_nan();
    const int64_t at = (int64_t)b * a.H + h;
    if (parts == 1) {
      const float o = n == 0 && !bad ? 0.0f : sum / all;
      store_as((T*)a.out + at * D + d, o);
    } else {
      a.part[(at * a.splits + split) * D + d] = sum;
    }
    if (d == 0 && a.ml != nullptr) a.ml[at * a.splits + split] = make_float2(top, all);
  }

  if (has_new && hblk == 0 && split == parts - 1) {
    const int at = __ldg(row + (n - 1) / a.c.page_size), in = (n - 1) % a.c.page_size;
    if (at >= 0 && at < a.c.pages) {
      T* kd = (T*)(a.c.k + (int64_t)at * a.c.k_page + (int64_t)in * a.c.k_slot + (int64_t)kvh * a.c.k_head);
      T* vd = (T*)(a.c.v + (int64_t)at * a.c.v_page + (int64_t)in * a.c.v_slot + (int64_t)kvh * a.c.v_head);
      for (int d = threadIdx.x; d < D; d += ATT_WARPS * 32) {
        kd[d] = ((const T*)knew)[d];
        vd[d] = ((const T*)vnew)[d];
      }
    }
  }
}

// Joins the splits of a row, and adds the weights to `mass`.  Blocks [0, B * H) join, the
// others take MASS_SLOTS slots of a key head each.

template <typename T>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedAttentionArgs a, int joins) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float2 stat[64];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < joins) {
    const int64_t at = blockIdx.x;
    const int n = max(0, min(__ldg(a.lengths + at / a.H), a.capacity));
    const int parts = paged_splits(n, a.splits, a.unit);
    if (parts == 1) return;                  // already whole
    const float2* ml = a.ml + at * a.splits;
    float top = neg_inf();
    for (int s = 0; s < parts; ++s) top = fmaxf(top, ml[s].x);
    for (int d = tid; d < a.c.channels; d += 128) {
      float sum = 0.0f, all = 0.0f;
      for (int s = 0; s < parts; ++s) {
        const float2 x = ml[s];
        const float f = x.x == neg_inf() ? 0.0f : tp_ex2(x.x - top);
        all += x.y * f;
        sum += a.part[(at * a.splits + s) * a.c.channels + d] * f;
      }
      store_as((T*)a.out + at * a.c.channels + d, sum / all);
    }
    return;
  }
  const int chunks = (a.capacity + MASS_SLOTS - 1) / MASS_SLOTS;
  const int i = blockIdx.x - joins, chunk = i % chunks, kvh = i / chunks % a.c.heads,
            b = i / chunks / a.c.heads;
  const int given = __ldg(a.lengths + b), n = max(0, min(given, a.capacity));
  if (chunk * MASS_SLOTS >= n) return;
  const int parts = paged_splits(n, a.splits, a.unit);
  const int64_t head = (int64_t)b * a.H + (int64_t)kvh * a.group;
  constexpr int PER = MASS_SLOTS / 128;
  float sum[PER] = {};
  for (int g0 = 0; g0 < a.group; g0 += 64) {
    const int some = min(64, a.group - g0);
    __syncthreads();
    if (tid < some) {
      const float2* ml = a.ml + (head + g0 + tid) * a.splits;
      float top = neg_inf(), all = 0.0f;
      for (int s = 0; s < parts; ++s) top = fmaxf(top, ml[s].x);
      for (int s = 0; s < parts; ++s) all += ml[s].y * (ml[s].x == neg_inf() ? 0.0f : tp_ex2(ml[s].x - top));
      stat[tid] = make_float2(top, 1.0f / all);
    }
    __syncthreads();
    for (int g = 0; g < some; ++g) {
      const float* sc = a.scores + (head + g0 + g) * a.capacity + chunk * MASS_SLOTS;
      const float2 st = stat[g];
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (chunk * MASS_SLOTS + k * 128 + tid < n) sum[k] += tp_ex2(sc[k * 128 + tid] - st.x) * st.y;
    }
  }
  float* mass = a.mass + (int64_t)b * a.mass_sb + (int64_t)kvh * a.mass_sh;
  const int fresh = a.key != nullptr && given == n ? n - 1 : -1;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int slot = chunk * MASS_SLOTS + k * 128 + tid;
    if (slot < n) mass[slot] = slot == fresh ? sum[k] : mass[slot] + sum[k];
  }
}

template <typename T, int LPK, int NCH, int G, bool GATED, bool VEC>
int attend(const PagedAttentionArgs& a, cudaStream_t stream) {
  constexpr int STAGES = NCH > 1 ? 2 : 3;
  using P = PagedAttend<T, LPK, NCH, G, GATED, VEC, STAGES>;
  auto* kernel = paged_attend_kernel<T, LPK, NCH, G, GATED, VEC, STAGES>;
  int st = allow_smem((const void*)kernel, P::SMEM);
  if (st != TP_OK) return st;
  const int64_t blocks = (int64_t)a.B * a.c.heads * a.head_blocks * a.splits;
  kernel<<<(unsigned)blocks, ATT_WARPS * 32, P::SMEM, stream>>>(a);
  return launch_status();
}

template <typename T>
int join(const PagedAttentionArgs& a, cudaStream_t stream) {
  const int joins = a.splits > 1 ? a.B * a.H : 0;
  int64_t blocks = joins;
  if (a.mass) blocks += (int64_t)a.B * a.c.heads * ceil_div(a.capacity, MASS_SLOTS);
  if (blocks == 0) return TP_OK;
  TP_RETURN_IF(blocks > INT32_MAX, TP_ERR_TOO_LARGE);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  // its blocks may be placed while the first kernel's last ones run; they wait for its end
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, paged_join_kernel<T>, a, joins));
}

// One query head at a time, two, or four: registers hold no more of their channels and sums.
template <typename T, int LPK, int NCH, bool VEC>
int attend_by_group(PagedAttentionArgs& a, cudaStream_t stream) {
  const bool gated = a.gate != nullptr;
  a.head_blocks = !VEC || a.group <= 2 ? (VEC ? 1 : a.group) : (a.group + 3) / 4;
  if constexpr (!VEC) {
    return gated ? attend<T, LPK, NCH, 1, true, false>(a, stream)
                 : attend<T, LPK, NCH, 1, false, false>(a, stream);
  } else {
    if (a.group == 1)
      return gated ? attend<T, LPK, NCH, 1, true, true>(a, stream)
                   : attend<T, LPK, NCH, 1, false, true>(a, stream);
    if (a.group == 2)
      return gated ? attend<T, LPK, NCH, 2, true, true>(a, stream)
                   : attend<T, LPK, NCH, 2, false, true>(a, stream);
    return gated ? attend<T, LPK, NCH, 4, true, true>(a, stream)
                 : attend<T, LPK, NCH, 4, false, true>(a, stream);
  }
}

}  // namespace

}  // namespace tp
