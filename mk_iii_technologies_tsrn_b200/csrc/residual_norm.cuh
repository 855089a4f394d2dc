// residual_norm.cuh -- the kernels of residual_norm.cu, instantiated for rows of
// fp32 and bf16 channels in files of their own.
#pragma once

#include "maxplus_internal.cuh"
#include "rowvec.cuh"

namespace tp {

namespace {


constexpr int RN_MAX_WARPS = 16;
// rows this many apart begin at the same element of 16 bytes, whatever their length
constexpr int RN_RESIDUES = 8;


// Where a thread stands in its row: thread t of the team's G, D channels, and the
// row's first channel at element `shift` of its first 16 bytes.
struct Place {
  int t, G, D, shift;
};

// A thread's elements come in groups of PV: one vector of VEC channels, or for
// VEC == 1 two single channels a team's width apart; in registers they are pairs
// (packed fp32 arithmetic).
// SH: rows that begin inside 16 bytes.  The vectors lie on 16 bytes all the same, so
// the first and the last of a row hold channels of its neighbours: they are read (not
// behind the tensor), taken as zeros, and never written.
template <typename T, int VEC, bool SH>
struct Group {
  static constexpr int PV = VEC == 1 ? 2 : VEC;      // elements
  static constexpr int P2 = PV / 2;                  // pairs
  RowVec<T, VEC> r[VEC == 1 ? 2 : 1];

  // first channel of vector v
  __device__ __forceinline__ static int column(int v, const Place& L) {
    return (v * L.G + L.t) * VEC - (SH ? L.shift : 0);
  }
  // whether the group has channels (VEC > 1 without SH: all or none of them)
  __device__ __forceinline__ static bool any(int g, const Place& L) {
    return column(VEC == 1 ? 2 * g : g, L) < L.D;
  }
  // whether the vector reaches over an end of the row
  __device__ __forceinline__ static bool over(int g, const Place& L) {
    const int c = column(g, L);
    return c < 0 || c + VEC > L.D;
  }
  // tail: fewer than VEC elements of the tensor lie behind the row
  __device__ __forceinline__ void load(const T* row, int g, const Place& L, bool tail) {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = column(2 * g + k, L);
        r[k].zero();
        if (row != nullptr && c < L.D) r[k].load(row + c);
      }
    } else {
      const int c = column(g, L);
      r[0].zero();
      if (row == nullptr || c >= L.D) return;
      if constexpr (SH) {
        if (tail && c + VEC > L.D) {
          T e[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            e[i] = T{};
            if (c + i >= 0 && c + i < L.D) e[i] = row[c + i];
          }
          r[0].pack(e);
          return;
        }
      }
      r[0].load_stream(row + c);
    }
  }
  __device__ __forceinline__ void get(float2* f, int g, const Place& L) const {
    float e[PV];
    if constexpr (VEC == 1) {
      r[0].get(e);
      r[1].get(e + 1);
    } else {
      r[0].get(e);
    }
#pragma unroll
    for (int i = 0; i < P2; ++i) f[i] = make_float2(e[2 * i], e[2 * i + 1]);
    if (SH) trim(f, g, L);
  }
  // f without what lies past the row's ends
  __device__ __forceinline__ static void trim(float2* f, int g, const Place& L) {
    if constexpr (VEC == 1) {
      if (column(2 * g, L) >= L.D) f[0].x = 0.f;
      if (column(2 * g + 1, L) >= L.D) f[0].y = 0.f;
    } else if constexpr (SH) {
      if (!over(g, L)) return;
      const int c = column(g, L);
#pragma unroll
      for (int i = 0; i < P2; ++i) {
        if ((unsigned)(c + 2 * i) >= (unsigned)L.D) f[i].x = 0.f;
        if ((unsigned)(c + 2 * i + 1) >= (unsigned)L.D) f[i].y = 0.f;
      }
    }
  }
  __device__ __forceinline__ static void store(T* row, const float2* f, int g, const Place& L) {
    float e[PV];
#pragma unroll
    for (int i = 0; i < P2; ++i) {
      e[2 * i] = f[i].x;
      e[2 * i + 1] = f[i].y;
    }
    if constexpr (VEC == 1) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = column(2 * g + k, L);
        RowVec<T, 1> o;
        o.set(e + k);
        if (c < L.D) o.store(row + c);
      }
    } else {
      const int c = column(g, L);
      if (SH && over(g, L)) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          RowVec<T, 1> o;
          o.set(e + i);
          if ((unsigned)(c + i) < (unsigned)L.D) o.store(row + c + i);
        }
        return;
      }
      RowVec<T, VEC> o;
      o.set(e);
      o.store_stream(row + c);
    }
  }
  // the same channels of a parameter staged in shared memory (from the row's first
  // 16 bytes on)
  __device__ __forceinline__ static void params(const float* p, float2* f, int g,
                                                const Place& L) {
    const float4* q = reinterpret_cast<const float4*>(p + (g * L.G + L.t) * VEC);
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 v = q[i];
      f[2 * i] = make_float2(v.x, v.y);
      f[2 * i + 1] = make_float2(v.z, v.w);
    }
  }
  // or in global memory (fp32 or bf16 storage)
  __device__ __forceinline__ static void params(const void* p, int is_bf16, float2* f, int g,
                                                const Place& L) {
    if constexpr (VEC == 1) {
      float e[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = column(2 * g + k, L);
        if (c < L.D)
          e[k] = is_bf16 ? tp_bf16_to_f32(__ldg((const unsigned short*)p + c))
                         : __ldg((const float*)p + c);
      }
      f[0] = make_float2(e[0], e[1]);
    } else if (!is_bf16) {
      const float4* q = reinterpret_cast<const float4*>((const float*)p + column(g, L));
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) {
        const float4 v = __ldg(q + i);
        f[2 * i] = make_float2(v.x, v.y);
        f[2 * i + 1] = make_float2(v.z, v.w);
      }
    } else {
      RowVec<bf16_t, VEC> v;
      float e[VEC];
      v.load((const bf16_t*)p + column(g, L));
      v.get(e);
#pragma unroll
      for (int i = 0; i < P2; ++i) f[i] = make_float2(e[2 * i], e[2 * i + 1]);
    }
  }
  // column sums of this thread in shared memory: acc += f
  __device__ __forceinline__ static void add_to(float* acc, const float2* f, int g) {
    if constexpr (VEC == 1) {
      float2* q = reinterpret_cast<float2*>(acc) + g * blockDim.x + threadIdx.x;
      *q = tp_add2(*q, f[0]);
    } else {
      float4* q = reinterpret_cast<float4*>(acc);
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) {
        const int at = (g * (VEC / 4) + i) * blockDim.x + threadIdx.x;
        const float4 r = q[at];
        const float2 lo = tp_add2(make_float2(r.x, r.y), f[2 * i]);
        const float2 hi = tp_add2(make_float2(r.z, r.w), f[2 * i + 1]);
        q[at] = make_float4(lo.x, lo.y, hi.x, hi.y);
      }
    }
  }
  // where add_to keeps element i of group g of thread t (of a team of threads)
  __device__ __forceinline__ static int place(int g, int i, int thread) {
    if constexpr (VEC == 1) return (g * blockDim.x + thread) * 2 + i;
    else return ((g * (VEC / 4) + i / 4) * blockDim.x + thread) * 4 + (i & 3);
  }
  __device__ __forceinline__ static int channel(int g, int i, const Place& L) {
    return VEC == 1 ? column(2 * g + i, L) : column(g, L) + i;
  }
};

// vectors that rows with any shift reach over, and their elements
inline __host__ __device__ int shifted_vectors(int D, int vec) { return (D + 2 * vec - 2) / vec; }
inline __host__ __device__ int staged_size(int D, int vec) { return shifted_vectors(D, vec) * vec; }

// Where the rows' parameters come from: global memory in fp32 or bf16, staged as
// fp32 in shared memory, or global memory in fp32.
enum { RN_ANY = 0, RN_STAGED = 1, RN_F32 = 2 };
template <typename T, int VEC, int MODE, bool SH>
struct Param {
  const void* p;
  int bf16;
  __device__ __forceinline__ explicit operator bool() const { return p != nullptr; }
  // copies the parameter to `to` (moved on) with all threads of the block
  __device__ __forceinline__ void stage(float*& to, int D, int shift) {
    if constexpr (MODE == RN_STAGED) {
      if (p == nullptr) return;
      const int size = SH ? staged_size(D, VEC) : D;
      for (int e = threadIdx.x; e < size; e += blockDim.x) {
        const int c = SH ? e - shift : e;
        float v = 0.f;
        if (!SH || (unsigned)c < (unsigned)D)
          v = bf16 ? tp_bf16_to_f32(__ldg((const unsigned short*)p + c))
                   : __ldg((const float*)p + c);
        to[e] = v;
      }
      p = to;
      to += size;
    }
  }
  __device__ __forceinline__ void get(float2* f, int g, const Place& L) const {
    if constexpr (MODE == RN_STAGED) Group<T, VEC, SH>::params((const float*)p, f, g, L);
    else Group<T, VEC, SH>::params(p, MODE == RN_F32 ? 0 : bf16, f, g, L);
  }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// exp(-|g|) of a gate with the gate's sign: what the sigmoid and its complement
// are formed from, twice in the backward.  To fp32 accuracy for bf16 storage too:
// the parameter gradients are fp32 sums of it.
__device__ __forceinline__ float gate_exp(float g) { return copysignf(expf(-fabsf(g)), g); }
// sigmoid and 1 - sigmoid: the larger one is 1 / (1 + e), the smaller e / (1 + e)
__device__ __forceinline__ void gate_from(float signed_e, float& s, float& rest) {
  const float e = fabsf(signed_e);
  const float big = rcp_approx(1.0f + e);
  const float small = e * big;
  const bool pos = __float_as_int(signed_e) >= 0;
  s = pos ? big : small;
  rest = pos ? small : big;
}

// Sum of one value, or of two, over the G threads of a team (the same bits in
// every thread).  `slots`: [2][warps of the block] float2 in shared memory; the
// two halves alternate, so one barrier per call is enough.  (Teams of several warps
// have a block each: named barriers with a number in a register make the compiler
// reserve all 16, and an SM then holds four blocks.)
template <bool TWO>
__device__ __forceinline__ float2 team_sum(float a, float b, int G, float2* slots, int& half) {
  const int lane = threadIdx.x & 31;
  if (TWO) {
    // one exchange hands a to the lower half of the warp and b to the upper
    const bool low = lane < 16;
    a = (low ? a : b) + __shfl_xor_sync(0xffffffffu, low ? b : a, 16);
  } else {
    a += __shfl_xor_sync(0xffffffffu, a, 16);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if (G == 32) {
    if (!TWO) return make_float2(a, 0.f);
    return make_float2(__shfl_sync(0xffffffffu, a, 0), __shfl_sync(0xffffffffu, a, 16));
  }
  const int warp = threadIdx.x >> 5, wpt = G >> 5;      // the team is the block
  float* s = reinterpret_cast<float*>(slots + half * RN_MAX_WARPS);
  half ^= 1;
  float2 t = make_float2(0.f, 0.f);
  if (TWO) {
    if ((lane & 15) == 0) s[warp * 2 + (lane >> 4)] = a;
    __syncthreads();
    for (int w = 0; w < wpt; ++w) t = tp_add2(t, reinterpret_cast<const float2*>(s)[w]);
  } else {
    if (lane == 0) s[warp] = a;
    __syncthreads();
    for (int w = 0; w < wpt; ++w) t.x += s[w];
  }
  return t;
}

// Ask for a row in L2: the team's next one, while this one is worked on.  (INWARD: its
// whole 16-byte pieces, where it begins or ends inside of one.)
template <bool INWARD, typename T>
__device__ __forceinline__ void prefetch_row(const T* row, int D) {
  if (row == nullptr) return;
  uintptr_t from = (uintptr_t)row, to = (uintptr_t)(row + D);
  if (INWARD) {
    from = (from + 15) & ~(uintptr_t)15;
    to &= ~(uintptr_t)15;
    if (from >= to) return;
  }
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from),
               "r"((uint32_t)(to - from)));
}

// 1 / deviation of a row from the sum of squares
__device__ __forceinline__ float inv_dev(float sum, float inv_d, float eps) {
  return 1.0f / sqrtf(sum * inv_d + eps);
}

__device__ __forceinline__ float scalar_param(const void* p, int is_bf16) {
  return is_bf16 ? tp_bf16_to_f32(*(const uint16_t*)p) : *(const float*)p;
}

// TG: 32, teams of a warp, or 0: a team of a.group threads is the block.  PM: where
// parameters come from.  GATE, BN: whether there is a gate and a branch norm (2: see
// the arguments).  (Looked up per row, the flags, types and addresses were half of
// all instructions: 93 per element in the backward of a gated LayerNorm row against
// 70, and 351 against 261 us for 65536 x 640 fp32.)
template <typename T, int VEC, int NV, int TG, int PM, int GATE, int BN, bool SH, int MAXT>
__global__ void __launch_bounds__(MAXT) residual_norm_fwd_kernel(const ResNormArgs a) {
  using V = Group<T, VEC, SH>;
  using P = Param<T, VEC, PM, SH>;
  constexpr int NG = VEC == 1 ? NV / 2 : NV, P2 = V::P2;
  extern __shared__ __align__(16) float s_par[];
  __shared__ float2 slots[2 * RN_MAX_WARPS];
  int half = 0;
  const int G = TG > 0 ? TG : a.group;
  const int t = TG > 0 ? threadIdx.x % TG : threadIdx.x, team = TG > 0 ? threadIdx.x / TG : 0;
  const int teams = TG > 0 ? blockDim.x / TG : 1, D = (int)a.D, pb = a.params_bf16;
  const Place L{t, G, D, SH ? (int)(blockIdx.x % RN_RESIDUES) * D % VEC : 0};
  const bool has_gate = GATE == 2 ? a.gate != nullptr : GATE != 0;
  const bool branch_norm = BN == 2 ? a.branch_norm != 0 : BN != 0;
  P pw{a.w, pb}, pbias{a.b, pb}, psc{a.scale_mode == 2 ? a.scale : nullptr, pb}, pbw{a.bw, pb},
      pbb{a.bb, pb};
  {
    float* to = s_par;
    pw.stage(to, D, L.shift);
    pbias.stage(to, D, L.shift);
    psc.stage(to, D, L.shift);
    pbw.stage(to, D, L.shift);
    pbb.stage(to, D, L.shift);
    if (PM == RN_STAGED) __syncthreads();
  }
  const bool layer = a.rms == 0;
  const float inv_d = 1.0f / (float)D;
  const float one_scale = a.scale_mode == 1 ? scalar_param(a.scale, pb) : 1.0f;
  // SH: the grid is a multiple of RN_RESIDUES, and all rows of a block are alike modulo it
  const int64_t first = SH ? ((int64_t)(blockIdx.x / RN_RESIDUES) * teams + team) * RN_RESIDUES +
                                 blockIdx.x % RN_RESIDUES
                           : (int64_t)blockIdx.x * teams + team;
  for (int64_t row = first; row < a.rows; row += (int64_t)gridDim.x * teams) {
    const bool tail = SH && (a.rows - 1 - row) * D < VEC;
    const T* xr = (const T*)a.x + row * a.ldx;
    const T* br = (const T*)a.branch + row * a.ldb;
    const T* gr = has_gate ? (const T*)a.gate + row * a.ldg : nullptr;
    if (PM != RN_ANY && t == 0) {
      const int64_t next = (int64_t)gridDim.x * teams;
      if (row + next < a.rows) {
        prefetch_row<VEC * sizeof(T) != 16 || SH>(br + next * a.ldb, D);
        if (has_gate) prefetch_row<VEC * sizeof(T) != 16 || SH>(gr + next * a.ldg, D);
        prefetch_row<VEC * sizeof(T) != 16 || SH>(xr + next * a.ldx, D);
      }
    }
    V vx[NG], vb[NG], vg[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      vb[g].load(br, g, L, tail);
      if (has_gate) vg[g].load(gr, g, L, tail);
      vx[g].load(xr, g, L, tail);
    }
    float m1 = 0.f, r1 = 1.f;
    if (branch_norm) {
      if (layer) {
        float2 s = both(0.f);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float2 p[P2];
          vb[g].get(p, g, L);
#pragma unroll
          for (int i = 0; i < P2; ++i) s = tp_add2(s, p[i]);
        }
        m1 = team_sum<false>(s.x + s.y, 0.f, G, slots, half).x * inv_d;
      }
      float2 q = both(0.f);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        if (!V::any(g, L)) continue;
        float2 p[P2];
        vb[g].get(p, g, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_add2(p[i], both(-m1));
        V::trim(p, g, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) q = tp_fma2(p[i], p[i], q);
      }
      r1 = inv_dev(team_sum<false>(q.x + q.y, 0.f, G, slots, half).x, inv_d, a.eps);
    }
    float2 y[NG * P2], s = both(0.f);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float2* yg = y + g * P2;
      vx[g].get(yg, g, L);
      if (!V::any(g, L)) continue;
      float2 p[P2], f[P2];
      vb[g].get(p, g, L);
      if (branch_norm) {
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_mul2(tp_add2(p[i], both(-m1)), both(r1));
        if (pbw) {
          pbw.get(f, g, L);
#pragma unroll
          for (int i = 0; i < P2; ++i) p[i] = tp_mul2(p[i], f[i]);
        }
        if (pbb) {
          pbb.get(f, g, L);
#pragma unroll
          for (int i = 0; i < P2; ++i) p[i] = tp_add2(p[i], f[i]);
        }
      }
      if (has_gate) {
        vg[g].get(f, g, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) {
          float2 sg;
          float om;
          gate_from(gate_exp(f[i].x), sg.x, om);
          gate_from(gate_exp(f[i].y), sg.y, om);
          p[i] = tp_mul2(sg, p[i]);
        }
      }
      if (psc) {
        psc.get(f, g, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_mul2(f[i], p[i]);
      } else if (a.scale_mode == 1) {
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_mul2(both(one_scale), p[i]);
      }
      V::trim(p, g, L);
#pragma unroll
      for (int i = 0; i < P2; ++i) {
        yg[i] = tp_add2(yg[i], p[i]);
        s = tp_add2(s, yg[i]);
      }
      V::store((T*)a.y + row * a.D, yg, g, L);
    }
    if (a.n == nullptr) {
      if (a.stats && t == 0)
        reinterpret_cast<float4*>(a.stats)[row] = make_float4(m1, r1, 0.f, 1.f);
      continue;
    }
    float m2 = 0.f;
    if (layer) m2 = team_sum<false>(s.x + s.y, 0.f, G, slots, half).x * inv_d;
    float2 q = both(0.f);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (!V::any(g, L)) continue;
      float2* yg = y + g * P2;
#pragma unroll
      for (int i = 0; i < P2; ++i) yg[i] = tp_add2(yg[i], both(-m2));
      V::trim(yg, g, L);
#pragma unroll
      for (int i = 0; i < P2; ++i) q = tp_fma2(yg[i], yg[i], q);
    }
    const float r2 = inv_dev(team_sum<false>(q.x + q.y, 0.f, G, slots, half).x, inv_d, a.eps);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (!V::any(g, L)) continue;
      float2 f[P2], w[P2];
#pragma unroll
      for (int i = 0; i < P2; ++i) f[i] = tp_mul2(y[g * P2 + i], both(r2));
      if (pw) {
        pw.get(w, g, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) f[i] = tp_mul2(f[i], w[i]);
      }
      if (pbias) {
        pbias.get(w, g, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) f[i] = tp_add2(f[i], w[i]);
      }
      V::store((T*)a.n + row * a.D, f, g, L);
    }
    if (a.stats && t == 0)
      reinterpret_cast<float4*>(a.stats)[row] = make_float4(m1, r1, m2, r2);
  }
}

template <typename T, int VEC, int NV, int TG, int PM, int GATE, int BN, bool SH, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 128 ? 3 : 1)
    residual_norm_bwd_kernel(const ResNormBwdArgs g) {
  using V = Group<T, VEC, SH>;
  using P = Param<T, VEC, PM, SH>;
  constexpr int NG = VEC == 1 ? NV / 2 : NV, P2 = V::P2, E = VEC * NV;
  extern __shared__ __align__(16) float s_acc[];   // [sums][E][blockDim], then the parameters
  __shared__ float2 slots[2 * RN_MAX_WARPS];
  const ResNormArgs& a = g.f;
  int half = 0;
  const int G = TG > 0 ? TG : a.group;
  const int t = TG > 0 ? threadIdx.x % TG : threadIdx.x, team = TG > 0 ? threadIdx.x / TG : 0;
  const int teams = TG > 0 ? blockDim.x / TG : 1, D = (int)a.D, pb = a.params_bf16;
  const Place L{t, G, D, SH ? (int)(blockIdx.x % RN_RESIDUES) * D % VEC : 0};
  const bool layer = a.rms == 0;
  const float inv_d = 1.0f / (float)D;
  const float one_scale = a.scale_mode == 1 ? scalar_param(a.scale, pb) : 1.0f;
  const int plane = E * blockDim.x;
  const bool has_gate = GATE == 2 ? a.gate != nullptr : GATE != 0;
  const bool branch_norm = BN == 2 ? a.branch_norm != 0 : BN != 0;
  P pw{a.w, pb}, psc{a.scale_mode == 2 ? a.scale : nullptr, pb}, pbw{a.bw, pb}, pbb{a.bb, pb};
  {
    float* to = s_acc + g.sums * plane;
    pw.stage(to, D, L.shift);
    psc.stage(to, D, L.shift);
    pbw.stage(to, D, L.shift);
    pbb.stage(to, D, L.shift);
  }
  for (int e = threadIdx.x; e < g.sums * plane; e += blockDim.x) s_acc[e] = 0.f;
  __syncthreads();
  float* const acc_w = g.slot_w >= 0 ? s_acc + g.slot_w * plane : nullptr;
  float* const acc_b = g.slot_b >= 0 ? s_acc + g.slot_b * plane : nullptr;
  float* const acc_s = g.slot_s >= 0 ? s_acc + g.slot_s * plane : nullptr;
  float* const acc_bw = g.slot_bw >= 0 ? s_acc + g.slot_bw * plane : nullptr;
  float* const acc_bb = g.slot_bb >= 0 ? s_acc + g.slot_bb * plane : nullptr;
  double sum_scale = 0.0;    // of the single scale: a row in fp32, the rows in 64 bits

  // SH: the grid is a multiple of RN_RESIDUES, and all rows of a block are alike modulo it
  const int64_t first = SH ? ((int64_t)(blockIdx.x / RN_RESIDUES) * teams + team) * RN_RESIDUES +
                                 blockIdx.x % RN_RESIDUES
                           : (int64_t)blockIdx.x * teams + team;
  for (int64_t row = first; row < a.rows; row += (int64_t)gridDim.x * teams) {
    const bool tail = SH && (a.rows - 1 - row) * D < VEC;
    const T* xr = g.dn ? (const T*)a.x + row * a.ldx : nullptr;
    const T* br = (const T*)a.branch + row * a.ldb;
    const T* gr = has_gate ? (const T*)a.gate + row * a.ldg : nullptr;
    const T* dnr = g.dn ? (const T*)g.dn + row * a.D : nullptr;
    const T* dyr = g.dy ? (const T*)g.dy + row * a.D : nullptr;
    const float4 st = __ldg(reinterpret_cast<const float4*>(a.stats) + row);
    const float m1 = st.x, r1 = st.y, m2 = st.z, r2 = st.w;
    if (PM != RN_ANY && t == 0) {
      const int64_t next = (int64_t)gridDim.x * teams;
      if (row + next < a.rows) {
        prefetch_row<VEC * sizeof(T) != 16 || SH>(br + next * a.ldb, D);
        if (has_gate) prefetch_row<VEC * sizeof(T) != 16 || SH>(gr + next * a.ldg, D);
        if (xr) prefetch_row<VEC * sizeof(T) != 16 || SH>(xr + next * a.ldx, D);
        if (dnr) prefetch_row<VEC * sizeof(T) != 16 || SH>(dnr + next * a.D, D);
        if (dyr) prefetch_row<VEC * sizeof(T) != 16 || SH>(dyr + next * a.D, D);
      }
    }
    V vx[NG], vb[NG], vg[NG], vn[NG], vy[NG];
#pragma unroll
    for (int v = 0; v < NG; ++v) {
      vb[v].load(br, v, L, tail);
      if (has_gate) vg[v].load(gr, v, L, tail);
      vx[v].load(xr, v, L, tail);
      vn[v].load(dnr, v, L, tail);
      vy[v].load(dyr, v, L, tail);
    }
    // the branch, normalised where it has a norm (without its affine part)
    auto branch_of = [&](int v, float2* p) {
      vb[v].get(p, v, L);
      if (branch_norm) {
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_mul2(tp_add2(p[i], both(-m1)), both(r1));
        V::trim(p, v, L);
      }
    };
    auto affine = [&](int v, float2* p) {
      float2 f[P2];
      if (pbw) {
        pbw.get(f, v, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_mul2(p[i], f[i]);
      }
      if (pbb) {
        pbb.get(f, v, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_add2(p[i], f[i]);
      }
    };
    float2 ge[NG * P2];      // of the gate, see gate_exp
    float2 yh[NG * P2];      // the normalised residual stream
    float2 gn[NG * P2];      // gradient of yh
    float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int v = 0; v < NG; ++v) {
      if (!V::any(v, L)) continue;
      float2 *yv = yh + v * P2, *nv = gn + v * P2, *ev = ge + v * P2;
      if (has_gate) {
        vg[v].get(ev, v, L);
#pragma unroll
        for (int i = 0; i < P2; ++i)
          ev[i] = make_float2(gate_exp(ev[i].x), gate_exp(ev[i].y));
      }
      if (dnr == nullptr) continue;
      float2 p[P2], f[P2];
      branch_of(v, p);
      affine(v, p);
      if (has_gate) {
#pragma unroll
        for (int i = 0; i < P2; ++i) {
          float2 sg;
          float om;
          gate_from(ev[i].x, sg.x, om);
          gate_from(ev[i].y, sg.y, om);
          p[i] = tp_mul2(sg, p[i]);
        }
      }
      if (psc) {
        psc.get(f, v, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_mul2(f[i], p[i]);
      } else if (a.scale_mode == 1) {
#pragma unroll
        for (int i = 0; i < P2; ++i) p[i] = tp_mul2(both(one_scale), p[i]);
      }
      vx[v].get(yv, v, L);
      vn[v].get(nv, v, L);
#pragma unroll
      for (int i = 0; i < P2; ++i)
        yv[i] = tp_mul2(tp_add2(tp_add2(yv[i], p[i]), both(-m2)), both(r2));
      V::trim(yv, v, L);
      if (acc_b) V::add_to(acc_b, nv, v);
      if (acc_w) {
#pragma unroll
        for (int i = 0; i < P2; ++i) f[i] = tp_mul2(nv[i], yv[i]);
        V::add_to(acc_w, f, v);
      }
      if (pw) {
        pw.get(f, v, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) nv[i] = tp_mul2(nv[i], f[i]);
      }
#pragma unroll
      for (int i = 0; i < P2; ++i) {
        s1 = tp_add2(s1, nv[i]);
        s2 = tp_fma2(nv[i], yv[i], s2);
      }
    }
    float c1 = 0.f, c2 = 0.f;
    if (dnr) {
      const float2 r = team_sum<true>(s1.x + s1.y, s2.x + s2.y, G, slots, half);
      c1 = layer ? r.x * inv_d : 0.f;
      c2 = r.y * inv_d;
    }
    s1 = s2 = both(0.f);
    float2 row_scale = both(0.f);
#pragma unroll
    for (int v = 0; v < NG; ++v) {
      if (!V::any(v, L)) continue;
      float2* nv = gn + v * P2;
      float2 d[P2], aff[P2], phat[P2], f[P2], sg[P2];
      vy[v].get(d, v, L);
      if (dnr) {
#pragma unroll
        for (int i = 0; i < P2; ++i)
          d[i] = tp_fma2(both(r2), tp_fma2(yh[v * P2 + i], both(-c2), tp_add2(nv[i], both(-c1))),
                         d[i]);
        V::trim(d, v, L);
      }
      V::store((T*)g.dx + row * a.D, d, v, L);
      branch_of(v, phat);
#pragma unroll
      for (int i = 0; i < P2; ++i) aff[i] = phat[i];
      affine(v, aff);
      if (has_gate) {
        float2 k[P2];
#pragma unroll
        for (int i = 0; i < P2; ++i) {
          float2 om;
          gate_from(ge[v * P2 + i].x, sg[i].x, om.x);
          gate_from(ge[v * P2 + i].y, sg[i].y, om.y);
          const float2 u = tp_mul2(sg[i], aff[i]);       // the gated branch
          k[i] = tp_mul2(u, om);                         // its derivative by the gate
          aff[i] = u;
        }
        if (psc) {
          psc.get(f, v, L);
#pragma unroll
          for (int i = 0; i < P2; ++i) {
            aff[i] = tp_mul2(d[i], aff[i]);
            d[i] = tp_mul2(d[i], f[i]);
          }
          if (acc_s) V::add_to(acc_s, aff, v);
        } else if (a.scale_mode == 1) {
#pragma unroll
          for (int i = 0; i < P2; ++i) {
            row_scale = tp_fma2(d[i], aff[i], row_scale);
            d[i] = tp_mul2(d[i], both(one_scale));
          }
        }
#pragma unroll
        for (int i = 0; i < P2; ++i) k[i] = tp_mul2(d[i], k[i]);
        V::store((T*)g.dgate + row * a.D, k, v, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) d[i] = tp_mul2(d[i], sg[i]);
      } else if (psc) {
        psc.get(f, v, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) {
          aff[i] = tp_mul2(d[i], aff[i]);
          d[i] = tp_mul2(d[i], f[i]);
        }
        if (acc_s) V::add_to(acc_s, aff, v);
      } else if (a.scale_mode == 1) {
#pragma unroll
        for (int i = 0; i < P2; ++i) {
          row_scale = tp_fma2(d[i], aff[i], row_scale);
          d[i] = tp_mul2(d[i], both(one_scale));
        }
      }
      if (!branch_norm) {
        V::store((T*)g.dbranch + row * a.D, d, v, L);
        continue;
      }
      if (acc_bb) V::add_to(acc_bb, d, v);
      if (acc_bw) {
#pragma unroll
        for (int i = 0; i < P2; ++i) f[i] = tp_mul2(d[i], phat[i]);
        V::add_to(acc_bw, f, v);
      }
      if (pbw) {
        pbw.get(f, v, L);
#pragma unroll
        for (int i = 0; i < P2; ++i) d[i] = tp_mul2(d[i], f[i]);
      }
#pragma unroll
      for (int i = 0; i < P2; ++i) {
        nv[i] = d[i];
        s1 = tp_add2(s1, d[i]);
        s2 = tp_fma2(d[i], phat[i], s2);
      }
    }
    sum_scale += (double)(row_scale.x + row_scale.y);
    if (branch_norm) {
      const float2 r = team_sum<true>(s1.x + s1.y, s2.x + s2.y, G, slots, half);
      c1 = layer ? r.x * inv_d : 0.f;
      c2 = r.y * inv_d;
#pragma unroll
      for (int v = 0; v < NG; ++v) {
        if (!V::any(v, L)) continue;
        float2 d[P2], phat[P2];
        branch_of(v, phat);
#pragma unroll
        for (int i = 0; i < P2; ++i)
          d[i] = tp_mul2(both(r1),
                         tp_fma2(phat[i], both(-c2), tp_add2(gn[v * P2 + i], both(-c1))));
        V::store((T*)g.dbranch + row * a.D, d, v, L);
      }
    }
  }
  // this block's column sums: its teams in order
  __syncthreads();
  const int64_t width = (int64_t)g.sums * a.D + 2;
  float* part = g.part + (int64_t)blockIdx.x * width;
  if (team == 0) {
    for (int k = 0; k < g.sums; ++k) {
#pragma unroll
      for (int v = 0; v < NG; ++v) {
#pragma unroll
        for (int i = 0; i < V::PV; ++i) {
          const int c = V::channel(v, i, L);
          if (c < 0 || c >= D) continue;
          float s = 0.f;
          for (int j = 0; j < teams; ++j) s += s_acc[k * plane + V::place(v, i, j * G + t)];
          part[(int64_t)k * a.D + c] = s;
        }
      }
    }
  }
  // and its share of the single scale's gradient, as two floats
  __shared__ double s_scale[RN_MAX_WARPS];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum_scale += __shfl_xor_sync(0xffffffffu, sum_scale, o);
  if ((threadIdx.x & 31) == 0) s_scale[threadIdx.x >> 5] = sum_scale;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += s_scale[w];
    const float hi = (float)s;
    part[width - 2] = hi;
    part[width - 1] = isinf(hi) ? 0.f : (float)(s - (double)hi);
  }
}

// Vector width and vectors per thread: of teams of one warp, of teams that are a
// block, and of both for rows that begin inside 16 bytes.
#define RN_WARP_F32(X) X(4, 1) X(4, 2) X(4, 3) X(4, 4) X(4, 5)
#define RN_BLOCK_F32(X) X(4, 4)
#define RN_WARP_BF16(X) X(8, 1) X(8, 2) X(8, 3)
#define RN_BLOCK_BF16(X) X(8, 2) X(4, 4)
#define RN_SHIFT_WARP_F32(X) X(4, 1) X(4, 3) X(4, 5)
#define RN_SHIFT_WARP_BF16(X) X(8, 1) X(8, 3)

template <typename T, int VEC, int NV, int TG, int PM, int GATE, int BN, bool SH>
int launch_fwd_kernel(const ResNormArgs& a, size_t smem, cudaStream_t stream) {
  constexpr int MAXT = TG == 32 ? 128 : 512;
  auto* kernel = residual_norm_fwd_kernel<T, VEC, NV, TG, PM, GATE, BN, SH, MAXT>;
  const int threads = TG == 32 ? 128 : a.group;
  if (smem > 40 * 1024) {
    const int st = allow_smem((const void*)kernel, smem);
    if (st != TP_OK) return st;
  }
  const int64_t want = ceil_div(a.rows, (int64_t)(threads / a.group));
  const int64_t cap = (int64_t)num_sms() * (2048 / threads < 32 ? 2048 / threads : 32);
  int64_t blocks = want < cap ? want : cap;
  if (SH) blocks = want < cap ? ceil_div(want, (int64_t)RN_RESIDUES) * RN_RESIDUES
                              : cap / RN_RESIDUES * RN_RESIDUES;
  kernel<<<(unsigned)blocks, threads, smem, stream>>>(a);
  return launch_status();
}

template <typename T, int VEC, int NV, int TG, int PM, int GATE, int BN, bool SH>
int launch_bwd_kernel(const ResNormBwdArgs& g, size_t smem, int blocks, cudaStream_t stream) {
  constexpr int MAXT = TG == 32 ? 128 : 512;
  auto* kernel = residual_norm_bwd_kernel<T, VEC, NV, TG, PM, GATE, BN, SH, MAXT>;
  if (smem > 40 * 1024) {
    const int st = allow_smem((const void*)kernel, smem);
    if (st != TP_OK) return st;
  }
  kernel<<<(unsigned)blocks, TG == 32 ? 128 : g.f.group, smem, stream>>>(g);
  return launch_status();
}

// the instantiation for the arguments' gate and branch norm
template <typename T, int VEC, int NV, int TG, int PM, bool SH>
int launch_fwd_known(const ResNormArgs& a, size_t smem, cudaStream_t s) {
  if (a.gate)
    return a.branch_norm ? launch_fwd_kernel<T, VEC, NV, TG, PM, 1, 1, SH>(a, smem, s)
                         : launch_fwd_kernel<T, VEC, NV, TG, PM, 1, 0, SH>(a, smem, s);
  return a.branch_norm ? launch_fwd_kernel<T, VEC, NV, TG, PM, 0, 1, SH>(a, smem, s)
                       : launch_fwd_kernel<T, VEC, NV, TG, PM, 0, 0, SH>(a, smem, s);
}
template <typename T, int VEC, int NV, int TG, int PM, bool SH>
int launch_bwd_known(const ResNormBwdArgs& g, size_t smem, int blocks, cudaStream_t s) {
  if (g.f.gate)
    return g.f.branch_norm ? launch_bwd_kernel<T, VEC, NV, TG, PM, 1, 1, SH>(g, smem, blocks, s)
                           : launch_bwd_kernel<T, VEC, NV, TG, PM, 1, 0, SH>(g, smem, blocks, s);
  return g.f.branch_norm ? launch_bwd_kernel<T, VEC, NV, TG, PM, 0, 1, SH>(g, smem, blocks, s)
                         : launch_bwd_kernel<T, VEC, NV, TG, PM, 0, 0, SH>(g, smem, blocks, s);
}

}  // namespace

// residual_norm_f32_*.cu, residual_norm_bf16_*.cu; shift: rows begin inside 16 bytes
int launch_residual_norm_fwd_f32(int vec, int nv, const ResNormArgs& a, size_t smem,
                                 cudaStream_t s);
int launch_residual_norm_bwd_f32(int vec, int nv, const ResNormBwdArgs& g, size_t smem,
                                 int blocks, cudaStream_t s);
int launch_residual_norm_fwd_bf16(int vec, int nv, const ResNormArgs& a, size_t smem,
                                  cudaStream_t s);
int launch_residual_norm_bwd_bf16(int vec, int nv, const ResNormBwdArgs& g, size_t smem,
                                  int blocks, cudaStream_t s);
int launch_residual_norm_fwd_shift(int nv, const ResNormArgs& a, size_t smem, cudaStream_t s);
int launch_residual_norm_bwd_shift_f32(int nv, const ResNormBwdArgs& g, size_t smem, int blocks,
                                       cudaStream_t s);
int launch_residual_norm_bwd_shift_bf16(int nv, const ResNormBwdArgs& g, size_t smem, int blocks,
                                        cudaStream_t s);

}  // namespace tp
