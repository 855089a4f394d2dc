// residual_norm.cu -- the residual stream between two blocks in one pass over
// it: the branch's own norm (optional), its sigmoid gate (optional), the
// residual scale (optional: one learnt number, or one of each channel), the
// residual sum, and the norm in front of the next block:
//
//   p = N(branch) * bw + bb              (or branch)
//   t = sigmoid(gate) * p                (or p)
//   y = x + scale * t                    the residual stream
//   n = N(y) * w + b                     what the next block reads
//
// N(v) = (v - mean(v)) / sqrt(var(v) + eps) (LayerNorm) or v / sqrt(mean(v^2)
// + eps) (RMS).  It is the step `x = x + branch(ln(x))` of the TSRN block
// (research/tsrn_dml.py:1096-1106) with the gate and mix of TropicalSSM
// (:975-980) and the next LayerNorm folded in.
//
// Both directions are bound by memory: the forward reads x, branch, gate once
// and writes y and n; the backward reads x, branch, gate, dy, dn once and
// writes dx, dbranch, dgate.  A team of G threads (a warp, or up to 16 warps
// for long rows) holds a whole row in registers, so the statistics cost no
// second read; all loads of a row are issued before the first use.  The
// backward recomputes y from x (the same bytes as reading y, and exact where
// the stored y is rounded to bf16) and takes the row statistics (mean and
// 1 / deviation of y and branch) from the forward.
//
// Parameter gradients are column sums.  Up to five of them run at once (w, b,
// channel scale, bw, bb), too many to stay in registers beside the row, so
// each thread keeps those of its own columns in shared memory (16-byte
// read-add-writes without conflicts, no synchronisation); a block adds its
// teams in order and a second kernel adds the blocks in order, so the same
// inputs give the same bits.
#include <initializer_list>

#include "maxplus_internal.cuh"
#include "rowvec.cuh"

namespace tp {

namespace {

constexpr int RN_MAX_WARPS = 16;

// VEC consecutive parameters (fp32 or bf16 storage) as fp32
template <int VEC>
__device__ __forceinline__ void load_params(const void* p, int is_bf16, int64_t c, float* f) {
  if (!is_bf16) {
    const float* q = static_cast<const float*>(p) + c;
    if constexpr (VEC == 1) {
      f[0] = __ldg(q);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(q + i));
        f[i] = t.x; f[i + 1] = t.y; f[i + 2] = t.z; f[i + 3] = t.w;
      }
    }
  } else {
    RowVec<bf16_t, VEC> r;
    r.load(static_cast<const bf16_t*>(p) + c);
    r.get(f);
  }
}

// Sum of two values over the G threads of a team (the same bits in every
// thread).  `slots`: [2][warps of the block] float2 in shared memory; the two
// halves alternate, so one barrier per call is enough.
__device__ __forceinline__ float2 team_sum(float a, float b, int G, float2* slots, int& half) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (G == 32) return make_float2(a, b);
  const int warp = threadIdx.x >> 5, wpt = G >> 5, team = warp / wpt;
  float2* s = slots + half * RN_MAX_WARPS;
  if ((threadIdx.x & 31) == 0) s[warp] = make_float2(a, b);
  asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(G) : "memory");
  half ^= 1;
  float2 t = s[team * wpt];
  for (int w = 1; w < wpt; ++w) {
    const float2 v = s[team * wpt + w];
    t.x += v.x;
    t.y += v.y;
  }
  return t;
}

template <typename T, int VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) residual_norm_fwd_kernel(const ResNormArgs a) {
  constexpr int E = VEC * NV;
  using V = RowVec<T, VEC>;
  __shared__ float2 slots[2 * RN_MAX_WARPS];
  int half = 0;
  const int G = a.group, t = threadIdx.x % G, team = threadIdx.x / G;
  const int teams = blockDim.x / G;
  const bool layer = a.rms == 0;
  const float inv_d = 1.0f / (float)a.D;
  const float one_scale =
      (a.scale_mode == 1) ? (a.params_bf16 ? tp_bf16_to_f32(*(const uint16_t*)a.scale)
                                           : *(const float*)a.scale)
                          : 1.0f;
  for (int64_t row = (int64_t)blockIdx.x * teams + team; row < a.rows;
       row += (int64_t)gridDim.x * teams) {
    const T* xr = (const T*)a.x + row * a.ldx;
    const T* br = (const T*)a.branch + row * a.ldb;
    const T* gr = a.gate ? (const T*)a.gate + row * a.ldg : nullptr;
    V vx[NV], vb[NV], vg[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c < a.D) {
        vx[v].load_stream(xr + c);
        vb[v].load_stream(br + c);
        if (gr) vg[v].load_stream(gr + c);
      } else {
        vx[v].zero();
        vb[v].zero();
      }
      if (!gr || c >= a.D) vg[v].zero();
    }
    float p[E], y[E];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      vb[v].get(p + v * VEC);
      vx[v].get(y + v * VEC);
    }
    float m1 = 0.f, r1 = 1.f;
    if (a.branch_norm) {
      if (layer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += p[i];
        m1 = team_sum(s, 0.f, G, slots, half).x * inv_d;
      }
      float q = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if ((v * G + t) * VEC < a.D)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float d = p[v * VEC + i] - m1;
            q += d * d;
          }
      r1 = 1.0f / sqrtf(team_sum(q, 0.f, G, slots, half).x * inv_d + a.eps);
    }
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c >= a.D) continue;
      float f[VEC], w[VEC];
      if (a.branch_norm) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[v * VEC + i] = (p[v * VEC + i] - m1) * r1;
        if (a.bw) {
          load_params<VEC>(a.bw, a.params_bf16, c, w);
#pragma unroll
          for (int i = 0; i < VEC; ++i) p[v * VEC + i] *= w[i];
        }
        if (a.bb) {
          load_params<VEC>(a.bb, a.params_bf16, c, w);
#pragma unroll
          for (int i = 0; i < VEC; ++i) p[v * VEC + i] += w[i];
        }
      }
      if (gr) {
        vg[v].get(f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float sg, om;
          sigmoid_pair(f[i], sg, om);
          p[v * VEC + i] = __fmul_rn(sg, p[v * VEC + i]);
        }
      }
      // products and the residual sum are rounded one by one, as the
      // unfused expression rounds them
      if (a.scale_mode == 2) {
        load_params<VEC>(a.scale, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[v * VEC + i] = __fmul_rn(w[i], p[v * VEC + i]);
      } else if (a.scale_mode == 1) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[v * VEC + i] = __fmul_rn(one_scale, p[v * VEC + i]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        y[v * VEC + i] = __fadd_rn(y[v * VEC + i], p[v * VEC + i]);
        s += y[v * VEC + i];
      }
      V o;
      o.set(y + v * VEC);
      o.store((T*)a.y + row * a.D + c);
    }
    if (a.n == nullptr) {
      if (a.stats && t == 0)
        reinterpret_cast<float4*>(a.stats)[row] = make_float4(m1, r1, 0.f, 1.f);
      continue;
    }
    float m2 = 0.f;
    if (layer) m2 = team_sum(s, 0.f, G, slots, half).x * inv_d;
    float q = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if ((v * G + t) * VEC < a.D)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = y[v * VEC + i] - m2;
          q += d * d;
        }
    const float r2 = 1.0f / sqrtf(team_sum(q, 0.f, G, slots, half).x * inv_d + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c >= a.D) continue;
      float f[VEC], w[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = (y[v * VEC + i] - m2) * r2;
      if (a.w) {
        load_params<VEC>(a.w, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] *= w[i];
      }
      if (a.b) {
        load_params<VEC>(a.b, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] += w[i];
      }
      V o;
      o.set(f);
      o.store((T*)a.n + row * a.D + c);
    }
    if (a.stats && t == 0)
      reinterpret_cast<float4*>(a.stats)[row] = make_float4(m1, r1, m2, r2);
  }
}

// acc[0..VEC) += f, one thread's slice of a column-sum array in shared memory
template <int VEC>
__device__ __forceinline__ void acc_add(float* acc, int v, const float* f) {
  if constexpr (VEC == 1) {
    acc[v * blockDim.x + threadIdx.x] += f[0];
  } else {
    float4* q = reinterpret_cast<float4*>(acc);
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const int at = (v * (VEC / 4) + i) * blockDim.x + threadIdx.x;
      float4 r = q[at];
      r.x += f[4 * i]; r.y += f[4 * i + 1]; r.z += f[4 * i + 2]; r.w += f[4 * i + 3];
      q[at] = r;
    }
  }
}

template <typename T, int VEC, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 128 ? 3 : 1)
    residual_norm_bwd_kernel(const ResNormBwdArgs g) {
  constexpr int E = VEC * NV;
  using V = RowVec<T, VEC>;
  extern __shared__ __align__(16) float s_acc[];   // [sums][E][blockDim]
  __shared__ float2 slots[2 * RN_MAX_WARPS];
  const ResNormArgs& a = g.f;
  int half = 0;
  const int G = a.group, t = threadIdx.x % G, team = threadIdx.x / G;
  const int teams = blockDim.x / G;
  const bool layer = a.rms == 0;
  const float inv_d = 1.0f / (float)a.D;
  const float one_scale =
      (a.scale_mode == 1) ? (a.params_bf16 ? tp_bf16_to_f32(*(const uint16_t*)a.scale)
                                           : *(const float*)a.scale)
                          : 1.0f;
  const int plane = E * blockDim.x;
  for (int k = 0; k < g.sums; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) s_acc[k * plane + e * blockDim.x + threadIdx.x] = 0.f;
  // (each thread clears and later adds to words of its own only up to the
  // block-wide barrier at the end: the two index maps differ, so wait here)
  __syncthreads();
  float* const acc_w = g.slot_w >= 0 ? s_acc + g.slot_w * plane : nullptr;
  float* const acc_b = g.slot_b >= 0 ? s_acc + g.slot_b * plane : nullptr;
  float* const acc_s = g.slot_s >= 0 ? s_acc + g.slot_s * plane : nullptr;
  float* const acc_bw = g.slot_bw >= 0 ? s_acc + g.slot_bw * plane : nullptr;
  float* const acc_bb = g.slot_bb >= 0 ? s_acc + g.slot_bb * plane : nullptr;
  float sum_scale = 0.f;

  for (int64_t row = (int64_t)blockIdx.x * teams + team; row < a.rows;
       row += (int64_t)gridDim.x * teams) {
    const T* xr = (const T*)a.x + row * a.ldx;
    const T* br = (const T*)a.branch + row * a.ldb;
    const T* gr = a.gate ? (const T*)a.gate + row * a.ldg : nullptr;
    const T* dnr = g.dn ? (const T*)g.dn + row * a.D : nullptr;
    const T* dyr = g.dy ? (const T*)g.dy + row * a.D : nullptr;
    const float4 st = __ldg(reinterpret_cast<const float4*>(a.stats) + row);
    const float m1 = st.x, r1 = st.y, m2 = st.z, r2 = st.w;
    V vx[NV], vb[NV], vg[NV], vn[NV], vy[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      const bool in = c < a.D;
      vx[v].zero(); vb[v].zero(); vg[v].zero(); vn[v].zero(); vy[v].zero();
      if (in) {
        if (dnr) {
          vx[v].load_stream(xr + c);
          vn[v].load_stream(dnr + c);
        }
        vb[v].load_stream(br + c);
        if (gr) vg[v].load_stream(gr + c);
        if (dyr) vy[v].load_stream(dyr + c);
      }
    }
    float p[E];      // the branch, normalised where it has a norm (without its affine part)
    float yh[E];     // the normalised residual stream
    float gn[E];     // gradient of yh
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      float* pv = p + v * VEC;
      float* yv = yh + v * VEC;
      float* nv = gn + v * VEC;
      vb[v].get(pv);
      vx[v].get(yv);
      vn[v].get(nv);
      if (c >= a.D) continue;
      float f[VEC], w[VEC];
      if (a.branch_norm) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) pv[i] = (pv[i] - m1) * r1;
      }
      if (dnr == nullptr) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = pv[i];
      if (a.bw) {
        load_params<VEC>(a.bw, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] *= w[i];
      }
      if (a.bb) {
        load_params<VEC>(a.bb, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] += w[i];
      }
      if (gr) {
        float gv[VEC];
        vg[v].get(gv);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float sg, om;
          sigmoid_pair(gv[i], sg, om);
          f[i] = __fmul_rn(sg, f[i]);
        }
      }
      if (a.scale_mode == 2) {
        load_params<VEC>(a.scale, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = __fmul_rn(w[i], f[i]);
      } else if (a.scale_mode == 1) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = __fmul_rn(one_scale, f[i]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) yv[i] = (__fadd_rn(yv[i], f[i]) - m2) * r2;
      if (acc_b) acc_add<VEC>(acc_b, v, nv);
      if (acc_w) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = nv[i] * yv[i];
        acc_add<VEC>(acc_w, v, f);
      }
      if (a.w) {
        load_params<VEC>(a.w, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) nv[i] *= w[i];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        s1 += nv[i];
        s2 += nv[i] * yv[i];
      }
    }
    float c1 = 0.f, c2 = 0.f;
    if (dnr) {
      const float2 r = team_sum(s1, s2, G, slots, half);
      c1 = layer ? r.x * inv_d : 0.f;
      c2 = r.y * inv_d;
    }
    s1 = s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c >= a.D) continue;
      float* pv = p + v * VEC;
      float* nv = gn + v * VEC;
      float d[VEC], w[VEC], aff[VEC], sg[VEC], om[VEC];
      vy[v].get(d);
      if (dnr) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[i] += r2 * (nv[i] - c1 - yh[v * VEC + i] * c2);
      }
      V o;
      o.set(d);
      o.store_stream((T*)g.dx + row * a.D + c);
      // the branch's affine value and the gate again (cheaper than keeping them)
#pragma unroll
      for (int i = 0; i < VEC; ++i) aff[i] = pv[i];
      if (a.bw) {
        load_params<VEC>(a.bw, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) aff[i] *= w[i];
      }
      if (a.bb) {
        load_params<VEC>(a.bb, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) aff[i] += w[i];
      }
      if (gr) {
        float gv[VEC];
        vg[v].get(gv);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sigmoid_pair(gv[i], sg[i], om[i]);
      }
      if (a.scale_mode != 0) {
        float f[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = d[i] * (gr ? sg[i] * aff[i] : aff[i]);
        if (a.scale_mode == 2) {
          if (acc_s) acc_add<VEC>(acc_s, v, f);
          load_params<VEC>(a.scale, a.params_bf16, c, w);
#pragma unroll
          for (int i = 0; i < VEC; ++i) d[i] *= w[i];
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            sum_scale += f[i];
            d[i] *= one_scale;
          }
        }
      }
      if (gr) {
        float f[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          f[i] = d[i] * aff[i] * (sg[i] * om[i]);
          d[i] *= sg[i];
        }
        o.set(f);
        o.store_stream((T*)g.dgate + row * a.D + c);
      }
      if (!a.branch_norm) {
        o.set(d);
        o.store_stream((T*)g.dbranch + row * a.D + c);
        continue;
      }
      if (acc_bb) acc_add<VEC>(acc_bb, v, d);
      if (acc_bw) {
        float f[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = d[i] * pv[i];
        acc_add<VEC>(acc_bw, v, f);
      }
      if (a.bw) {
        load_params<VEC>(a.bw, a.params_bf16, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[i] *= w[i];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        nv[i] = d[i];
        s1 += d[i];
        s2 += d[i] * pv[i];
      }
    }
    if (a.branch_norm) {
      const float2 r = team_sum(s1, s2, G, slots, half);
      c1 = layer ? r.x * inv_d : 0.f;
      c2 = r.y * inv_d;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * G + t) * VEC;
        if (c >= a.D) continue;
        float d[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          d[i] = r1 * (gn[v * VEC + i] - c1 - p[v * VEC + i] * c2);
        V o;
        o.set(d);
        o.store_stream((T*)g.dbranch + row * a.D + c);
      }
    }
  }
  // this block's column sums: its teams in order
  __syncthreads();
  const int64_t width = (int64_t)g.sums * a.D + 1;
  float* part = g.part + (int64_t)blockIdx.x * width;
  if (team == 0) {
    for (int k = 0; k < g.sums; ++k) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int c = (v * G + t) * VEC + i;
          if (c >= a.D) continue;
          const float* q;
          int step;
          if constexpr (VEC == 1) {
            q = s_acc + k * plane + v * blockDim.x + t;
            step = G;
          } else {
            q = s_acc + k * plane + ((v * (VEC / 4) + i / 4) * blockDim.x + t) * 4 + (i & 3);
            step = 4 * G;
          }
          float s = 0.f;
          for (int j = 0; j < teams; ++j) s += q[j * step];
          part[(int64_t)k * a.D + c] = s;
        }
      }
    }
  }
  // and its share of the single scale's gradient
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum_scale += __shfl_xor_sync(0xffffffffu, sum_scale, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5].x = sum_scale;
  __syncthreads();
  if (threadIdx.x == 0) {
    float s = 0.f;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += slots[w].x;
    part[width - 1] = s;
  }
}

// Column sums over the blocks' partials, in block order: 32 columns per block,
// 8 warps each take a contiguous range of the partials.
__global__ void __launch_bounds__(256) residual_norm_sum_kernel(const ResNormBwdArgs g,
                                                                int blocks) {
  __shared__ float s[8][32];
  const int64_t width = (int64_t)g.sums * g.f.D + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + lane;
  const int per = (blocks + 7) / 8;
  const int lo = warp * per, hi = min(blocks, lo + per);
  float acc = 0.f;
  if (col < width) {
#pragma unroll 8
    for (int i = lo; i < hi; ++i) acc += g.part[(int64_t)i * width + col];
  }
  s[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || col >= width) return;
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += s[w][lane];
  if (col == width - 1) {
    if (g.f.scale_mode == 1 && g.dscale) *g.dscale = t;
    return;
  }
  const int k = (int)(col / g.f.D);
  const int64_t c = col - (int64_t)k * g.f.D;
  if (k == g.slot_w) g.dw[c] = t;
  else if (k == g.slot_b) g.db[c] = t;
  else if (k == g.slot_s) g.dscale[c] = t;
  else if (k == g.slot_bw) g.dbw[c] = t;
  else if (k == g.slot_bb) g.dbb[c] = t;
}

struct Plan {
  int vec, nv, group;
};

// Team size and vectors per thread: the smallest cover of the row (fewest idle
// lanes), then the smallest team (fewer barriers).  nv is bounded by the
// registers of the backward (five row arrays).
bool plan_row(int vec, int64_t D, Plan& p) {
  const int nv_max = vec == 1 ? 16 : (vec == 8 ? 3 : 5);
  const int64_t n = ceil_div(D, (int64_t)vec);
  int64_t best = INT64_MAX;
  for (int G = 32; G <= 512; G *= 2) {
    int64_t nv = ceil_div(n, (int64_t)G);
    if (nv > nv_max) continue;
    if (vec == 1) nv = 16;
    if (G * nv < best) {
      best = G * nv;
      p = {vec, (int)nv, G};
    }
  }
  return best != INT64_MAX;
}

template <typename F>
int with_kernel(const Plan& p, bool bf16, F&& f) {
#define RN_CASE(T, VEC, NV)                         \
  if (p.vec == VEC && p.nv == NV) {                 \
    if (p.group <= 128) return f.template go<T, VEC, NV, 128>(); \
    return f.template go<T, VEC, NV, 512>();        \
  }
  if (!bf16) {
    RN_CASE(float, 4, 1)
    RN_CASE(float, 4, 2)
    RN_CASE(float, 4, 3)
    RN_CASE(float, 4, 4)
    RN_CASE(float, 4, 5)
    RN_CASE(float, 1, 16)
  } else {
    RN_CASE(bf16_t, 8, 1)
    RN_CASE(bf16_t, 8, 2)
    RN_CASE(bf16_t, 8, 3)
    RN_CASE(bf16_t, 4, 1)
    RN_CASE(bf16_t, 4, 2)
    RN_CASE(bf16_t, 4, 3)
    RN_CASE(bf16_t, 4, 4)
    RN_CASE(bf16_t, 4, 5)
    RN_CASE(bf16_t, 1, 16)
  }
#undef RN_CASE
  return TP_ERR_UNSUPPORTED;
}

int block_threads(const Plan& p) { return p.group < 128 ? 128 : p.group; }

struct FwdLaunch {
  const ResNormArgs& a;
  const Plan& p;
  cudaStream_t stream;
  template <typename T, int VEC, int NV, int MAXT>
  int go() {
    const int threads = block_threads(p), teams = threads / p.group;
    const int64_t want = ceil_div(a.rows, (int64_t)teams);
    const int64_t cap = (int64_t)num_sms() * (2048 / threads);
    residual_norm_fwd_kernel<T, VEC, NV, MAXT>
        <<<(unsigned)(want < cap ? want : cap), threads, 0, stream>>>(a);
    return launch_status();
  }
};

struct BwdLaunch {
  const ResNormBwdArgs& g;
  const Plan& p;
  cudaStream_t stream;
  template <typename T, int VEC, int NV, int MAXT>
  int go() {
    const int threads = block_threads(p);
    const size_t smem = (size_t)g.sums * VEC * NV * threads * sizeof(float);
    auto* kernel = residual_norm_bwd_kernel<T, VEC, NV, MAXT>;
    const cudaError_t e = cudaFuncSetAttribute(
        (const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return cuda_status(e);
    const int blocks = residual_norm_bwd_blocks(g.f.rows, g.f.D);
    kernel<<<(unsigned)blocks, threads, smem, stream>>>(g);
    const int64_t width = (int64_t)g.sums * g.f.D + 1;
    residual_norm_sum_kernel<<<(unsigned)ceil_div(width, (int64_t)32), 256, 0, stream>>>(g,
                                                                                      blocks);
    return launch_status();
  }
};

bool vec_ok(const ResNormArgs& a, int vec, int esize) {
  const int64_t m = (int64_t)vec * esize - 1;   // 8- or 16-byte vectors
  auto al = [&](const void* q) { return q == nullptr || (((uintptr_t)q) & m) == 0; };
  auto al16 = [](const void* q) { return q == nullptr || aligned16(q); };
  return a.D % vec == 0 && al(a.x) && al(a.branch) && al(a.gate) && al(a.y) && al(a.n) &&
         a.ldx % vec == 0 && a.ldb % vec == 0 && (a.gate == nullptr || a.ldg % vec == 0) &&
         al16(a.w) && al16(a.b) && al16(a.bw) && al16(a.bb) &&
         (a.scale_mode != 2 || al16(a.scale));
}

bool make_plan(const ResNormArgs& a, int align_of_grads, Plan& p) {
  const bool bf16 = a.dtype == TP_DTYPE_BF16;
  const int esize = bf16 ? 2 : 4;
  for (int vec : {bf16 ? 8 : 4, bf16 ? 4 : 1, 1}) {
    if (vec > 1 && (!vec_ok(a, vec, esize) || align_of_grads % (vec * esize) != 0)) continue;
    return plan_row(vec, a.D, p);
  }
  return false;
}

int common_align(std::initializer_list<const void*> ps) {
  uintptr_t m = 16;
  for (const void* q : ps) m |= (uintptr_t)q;
  return (int)(m & (~m + 1));
}

}  // namespace

bool residual_norm_supported(int64_t D) { return D >= 1 && D <= 8192; }

int residual_norm_bwd_blocks(int64_t rows, int64_t D) {
  // three blocks of 128 threads on each SM (one of 256 or 512), each with at
  // least one row of a team
  const int64_t per_sm = D > 2560 ? 1 : 3;
  const int64_t cap = (int64_t)num_sms() * per_sm;
  return (int)(rows < cap ? (rows > 0 ? rows : 1) : cap);
}

int launch_residual_norm_fwd(const ResNormArgs& args, cudaStream_t stream) {
  ResNormArgs a = args;
  Plan p;
  if (!make_plan(a, 16, p)) return TP_ERR_UNSUPPORTED;
  a.group = p.group;
  FwdLaunch l{a, p, stream};
  return with_kernel(p, a.dtype == TP_DTYPE_BF16, l);
}

int launch_residual_norm_bwd(const ResNormBwdArgs& args, cudaStream_t stream) {
  ResNormBwdArgs g = args;
  Plan p;
  if (!make_plan(g.f, common_align({g.dy, g.dn, g.dx, g.dbranch, g.dgate}), p))
    return TP_ERR_UNSUPPORTED;
  g.f.group = p.group;
  int k = 0;
  g.slot_w = g.dw ? k++ : -1;
  g.slot_b = g.db ? k++ : -1;
  g.slot_s = (g.f.scale_mode == 2 && g.dscale) ? k++ : -1;
  g.slot_bw = g.dbw ? k++ : -1;
  g.slot_bb = g.dbb ? k++ : -1;
  g.sums = k;
  BwdLaunch l{g, p, stream};
  return with_kernel(p, g.f.dtype == TP_DTYPE_BF16, l);
}

}  // namespace tp
