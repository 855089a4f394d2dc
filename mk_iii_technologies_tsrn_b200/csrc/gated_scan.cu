// gated_scan.cu -- the gated linear recurrence over [B, T, C] and its backward:
//
//   decay form:    h_t = a_t h_{t-1} + u_t            (gate = a, x = u)
//   sigmoid form:  f = sigmoid(gate_t);  h_t = f h_{t-1} + (1 - f) x_t
//
// the (plus, times) counterpart of the max-plus scan (scan.cu), with a gate of
// its own for every element.  States are fp32 whatever the storage; h is
// rounded once when it is stored.
//
// Steps compose: a run of steps maps h -> A h + H with A the product of its
// gates and H its result from a zero state.  One warp owns 32 lanes of channels
// (two bf16 channels per lane, so a row is 128 bytes either way) and L
// consecutive steps, all in registers; the W warps of a block own consecutive
// runs, and the S blocks of a thread-block cluster consecutive groups of those.
// An iteration loads S * W * L steps, forms every warp's (A, H), exchanges them
// through shared memory (between the cluster's blocks through distributed
// shared memory, one cluster barrier), applies the runs in order to the carried
// state, and runs each warp's steps again from its own starting state.  So the
// inputs are read once, the order of every operation is fixed (the same bits
// on each call), and few channels still spread over many SMs.
//
// The backward walks the iterations from the end with the mirrored recurrence
//   g_t = dh_t + c_{t+1},  c_t = a_t g_t   (c_t: gradient of h_{t-1})
// and forms da_t = g_t h_{t-1} from states it recomputes in fp32: the forward
// keeps one state per 64 steps.  It reads gate, x and dh once and writes dgate
// and dx: like the forward it is bound by memory.
#include "maxplus_internal.cuh"
#include "rowvec.cuh"

namespace tp {

namespace {

constexpr int GS_MAX_CLUSTER = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}

// store a pair into the same shared-memory place of the cluster's block `rank`
__device__ __forceinline__ void store_remote(float2* local, uint32_t rank, float2 v) {
  uint32_t dst;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(dst)
               : "r"(tp_smem_addr(local)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(v.x), "f"(v.y)
               : "memory");
}

// A h + H; a zero state stays H where the product of many gates overflowed
__device__ __forceinline__ float apply_run(float A, float H, float h) {
  return h == 0.0f ? H : fmaf(A, h, H);
}

// gate and input as the recurrence's a and u (and 1 - a in the sigmoid form)
template <int FORM>
__device__ __forceinline__ void gate_of(float z, float x, float& a, float& rest, float& u) {
  if constexpr (FORM == TP_GATE_SIGMOID) {
    sigmoid_pair(z, a, rest);
    u = rest * x;
  } else {
    a = z;
    rest = 1.0f;
    u = x;
  }
}

struct Where {
  int64_t b, c;       // batch row, this lane's first channel
  bool in;            // the lane has channels
  int64_t len;        // live steps of the row
  int rank;           // block of the cluster
};

template <int CPL>
__device__ __forceinline__ Where place(const GatedScanArgs& a, int S, int64_t tiles) {
  Where w;
  const int64_t id = blockIdx.x / S;
  w.rank = S > 1 ? (int)cluster_rank() : 0;
  w.b = id / tiles;
  w.c = (id - w.b * tiles) * (32 * CPL) + (threadIdx.x & 31) * CPL;
  w.in = w.c < a.C;
  w.len = a.T;
  if (a.lengths) {
    const int64_t n = a.lengths[w.b];
    w.len = n < 0 ? 0 : (n < a.T ? n : a.T);
  }
  return w;
}

template <typename T, int CPL, int FORM, int L, int W>
__global__ void __launch_bounds__(32 * W) gated_scan_fwd_kernel(const GatedScanArgs a,
                                                                const int S,
                                                                const int64_t tiles) {
  using V = RowVec<T, CPL>;
  __shared__ float2 s_run[2][W][32 * CPL];
  __shared__ float2 s_blk[2][GS_MAX_CLUSTER][32 * CPL];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Where w = place<CPL>(a, S, tiles);
  const T* gp = (const T*)a.gate + w.b * a.gate_sb + w.c;
  const T* xp = (const T*)a.x + w.b * a.x_sb + w.c;
  T* hp = (T*)a.h + (w.b * a.T) * a.C + w.c;
  const int64_t chunks = ceil_div(a.T, (int64_t)GATED_SCAN_CHUNK);
  const int64_t step = (int64_t)S * W * L;
  const int64_t iters = ceil_div(a.T, step);
  float carry[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k) carry[k] = (a.h0 && w.in) ? a.h0[w.b * a.C + w.c + k] : 0.0f;

  V vg[L], vx[L];
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (w.in && t0 + i < w.len) {
        vg[i].load_stream(gp + (t0 + i) * a.gate_st);
        vx[i].load_stream(xp + (t0 + i) * a.x_st);
      }
    }
  };
  if (S > 1) cluster_sync();   // every block of the cluster runs before the first remote store
  fetch(((int64_t)w.rank * W + warp) * L);
  for (int64_t it = 0; it < iters; ++it) {
    const int par = (int)(it & 1);
    const int64_t t0 = it * step + ((int64_t)w.rank * W + warp) * L;
    float A[L][CPL], U[L][CPL];
    float pa[CPL], ph[CPL];
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      pa[k] = 1.0f;
      ph[k] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float z[CPL], x[CPL], rest;
      vg[i].get(z);
      vx[i].get(x);
      const bool live = w.in && t0 + i < w.len;
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        gate_of<FORM>(z[k], x[k], A[i][k], rest, U[i][k]);
        if (!live) {            // past the end the state stays
          A[i][k] = 1.0f;
          U[i][k] = 0.0f;
        }
        ph[k] = fmaf(A[i][k], ph[k], U[i][k]);
        pa[k] *= A[i][k];
      }
    }
    if (it + 1 < iters) fetch(t0 + step);
#pragma unroll
    for (int k = 0; k < CPL; ++k) s_run[par][warp][lane * CPL + k] = make_float2(pa[k], ph[k]);
    __syncthreads();
    float mine[CPL];
    if (S == 1) {
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        float h = carry[k];
#pragma unroll
        for (int q = 0; q < W; ++q) {
          if (q == warp) mine[k] = h;
          const float2 r = s_run[par][q][lane * CPL + k];
          h = apply_run(r.x, r.y, h);
        }
        carry[k] = h;
      }
    } else {
      if (warp == 0) {
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          float2 r = s_run[par][0][lane * CPL + k];
#pragma unroll
          for (int q = 1; q < W; ++q) {
            const float2 n = s_run[par][q][lane * CPL + k];
            r.y = apply_run(n.x, n.y, r.y);
            r.x *= n.x;
          }
          for (int q = 0; q < S; ++q) store_remote(&s_blk[par][w.rank][lane * CPL + k], q, r);
        }
      }
      cluster_sync();
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        float h = carry[k], start = 0.0f;
        for (int q = 0; q < S; ++q) {
          if (q == w.rank) start = h;
          const float2 r = s_blk[par][q][lane * CPL + k];
          h = apply_run(r.x, r.y, h);
        }
        carry[k] = h;
        for (int q = 0; q < warp; ++q) {
          const float2 r = s_run[par][q][lane * CPL + k];
          start = apply_run(r.x, r.y, start);
        }
        mine[k] = start;
      }
    }
    if (a.states && w.in && t0 < a.T && (t0 % GATED_SCAN_CHUNK) == 0) {
#pragma unroll
      for (int k = 0; k < CPL; ++k)
        a.states[(w.b * chunks + t0 / GATED_SCAN_CHUNK) * a.C + w.c + k] = mine[k];
    }
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float o[CPL];
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        mine[k] = fmaf(A[i][k], mine[k], U[i][k]);
        o[k] = t0 + i < w.len ? mine[k] : 0.0f;
      }
      if (w.in && t0 + i < a.T) {
        V v;
        v.set(o);
        v.store_stream(hp + (t0 + i) * a.C);
      }
    }
  }
  if (a.h_last && w.rank == 0 && warp == 0 && w.in) {
#pragma unroll
    for (int k = 0; k < CPL; ++k) a.h_last[w.b * a.C + w.c + k] = carry[k];
  }
}

template <typename T, int CPL, int FORM, int L, int W>
__global__ void __launch_bounds__(32 * W) gated_scan_bwd_kernel(const GatedScanBwdArgs g,
                                                                const int S,
                                                                const int64_t tiles) {
  static_assert(GATED_SCAN_CHUNK % L == 0 && (W * L) % GATED_SCAN_CHUNK == 0, "");
  using V = RowVec<T, CPL>;
  const GatedScanArgs& a = g.f;
  __shared__ float2 s_run[2][W][32 * CPL];   // product of the gates, H forwards
  __shared__ float s_rev[2][W][32 * CPL];    // result of the run backwards
  __shared__ float2 s_blk[2][GS_MAX_CLUSTER][32 * CPL];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Where w = place<CPL>(a, S, tiles);
  const T* gp = (const T*)a.gate + w.b * a.gate_sb + w.c;
  const T* xp = (const T*)a.x + w.b * a.x_sb + w.c;
  const T* dp = g.dh ? (const T*)g.dh + (w.b * a.T) * a.C + w.c : nullptr;
  T* dgp = (T*)g.dgate + (w.b * a.T) * a.C + w.c;
  T* dxp = (T*)g.dx + (w.b * a.T) * a.C + w.c;
  const int64_t chunks = ceil_div(a.T, (int64_t)GATED_SCAN_CHUNK);
  const int64_t step = (int64_t)S * W * L;
  const int64_t iters = ceil_div(a.T, step);
  float carry[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k)
    carry[k] = (g.dh_last && w.in) ? g.dh_last[w.b * a.C + w.c + k] : 0.0f;

  V vg[L], vx[L], vd[L];
  float first[CPL];
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (w.in && t0 + i < w.len) {
        vg[i].load_stream(gp + (t0 + i) * a.gate_st);
        vx[i].load_stream(xp + (t0 + i) * a.x_st);
        if (dp) vd[i].load_stream(dp + (t0 + i) * a.C);
        else vd[i].zero();
      }
    }
  };
  if (S > 1) cluster_sync();   // every block of the cluster runs before the first remote store
  for (int64_t it = iters - 1; it >= 0; --it) {
    const int par = (int)(it & 1);
    const int64_t tb = it * step + (int64_t)w.rank * W * L;   // the block's first step
    const int64_t t0 = tb + warp * L;
    fetch(t0);
    // the state before this warp's 64-step chunk, and the chunk's first warp
    const int64_t chunk = t0 / GATED_SCAN_CHUNK;
    const int lead = warp - (int)((t0 % GATED_SCAN_CHUNK) / L);
#pragma unroll
    for (int k = 0; k < CPL; ++k)
      first[k] = (w.in && t0 < w.len) ? a.states[(w.b * chunks + chunk) * a.C + w.c + k] : 0.0f;
    float A[L][CPL], R[L][CPL], U[L][CPL], D[L][CPL];
    float pa[CPL], ph[CPL], pr[CPL];
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      pa[k] = 1.0f;
      ph[k] = pr[k] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float z[CPL], x[CPL];
      vg[i].get(z);
      vx[i].get(x);
      vd[i].get(D[i]);
      const bool live = w.in && t0 + i < w.len;
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        gate_of<FORM>(z[k], x[k], A[i][k], R[i][k], U[i][k]);
        if (!live) {
          A[i][k] = 1.0f;
          U[i][k] = 0.0f;
          D[i][k] = 0.0f;
        }
        ph[k] = fmaf(A[i][k], ph[k], U[i][k]);
        pa[k] *= A[i][k];
      }
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i)
#pragma unroll
      for (int k = 0; k < CPL; ++k) pr[k] = A[i][k] * (D[i][k] + pr[k]);
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      s_run[par][warp][lane * CPL + k] = make_float2(pa[k], ph[k]);
      s_rev[par][warp][lane * CPL + k] = pr[k];
    }
    __syncthreads();
    float mine[CPL];
    if (S == 1) {
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        float c = carry[k];
#pragma unroll
        for (int q = W - 1; q >= 0; --q) {
          if (q == warp) mine[k] = c;
          c = apply_run(s_run[par][q][lane * CPL + k].x, s_rev[par][q][lane * CPL + k], c);
        }
        carry[k] = c;
      }
    } else {
      if (warp == 0) {
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          float2 r = make_float2(s_run[par][W - 1][lane * CPL + k].x,
                                 s_rev[par][W - 1][lane * CPL + k]);
#pragma unroll
          for (int q = W - 2; q >= 0; --q) {
            const float n = s_run[par][q][lane * CPL + k].x;
            r.y = apply_run(n, s_rev[par][q][lane * CPL + k], r.y);
            r.x *= n;
          }
          for (int q = 0; q < S; ++q) store_remote(&s_blk[par][w.rank][lane * CPL + k], q, r);
        }
      }
      cluster_sync();
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        float c = carry[k], start = 0.0f;
        for (int q = S - 1; q >= 0; --q) {
          if (q == w.rank) start = c;
          const float2 r = s_blk[par][q][lane * CPL + k];
          c = apply_run(r.x, r.y, c);
        }
        carry[k] = c;
        for (int q = W - 1; q > warp; --q)
          start = apply_run(s_run[par][q][lane * CPL + k].x, s_rev[par][q][lane * CPL + k],
                            start);
        mine[k] = start;
      }
    }
    float before[L][CPL];      // h_{t-1}
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      float h = first[k];
      for (int q = lead; q < warp; ++q) {
        const float2 r = s_run[par][q][lane * CPL + k];
        h = apply_run(r.x, r.y, h);
      }
#pragma unroll
      for (int i = 0; i < L; ++i) {
        before[i][k] = h;
        h = fmaf(A[i][k], h, U[i][k]);
      }
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      float oz[CPL], ox[CPL];
      const bool live = t0 + i < w.len;
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        const float gr = D[i][k] + mine[k];
        mine[k] = A[i][k] * gr;
        if constexpr (FORM == TP_GATE_SIGMOID) {
          // d(f h + (1 - f) x)/dz = f (1 - f) (h - x) = f ((1 - f) h - u)
          oz[k] = gr * (A[i][k] * fmaf(R[i][k], before[i][k], -U[i][k]));
          ox[k] = gr * R[i][k];
        } else {
          oz[k] = gr * before[i][k];
          ox[k] = gr;
        }
        if (!live) oz[k] = ox[k] = 0.0f;
      }
      if (w.in && t0 + i < a.T) {
        V v;
        v.set(oz);
        v.store_stream(dgp + (t0 + i) * a.C);
        v.set(ox);
        v.store_stream(dxp + (t0 + i) * a.C);
      }
    }
  }
  if (g.dh0 && w.rank == 0 && warp == 0 && w.in) {
#pragma unroll
    for (int k = 0; k < CPL; ++k) g.dh0[w.b * a.C + w.c + k] = carry[k];
  }
}

// One step of every row, the state updated in place: a serving step.
template <typename T, int FORM>
__global__ void __launch_bounds__(256)
    gated_scan_step_kernel(int64_t B, int64_t C, const T* __restrict__ gate, int64_t ldg,
                           const T* __restrict__ x, int64_t ldx, float* state, int64_t lds,
                           T* h) {
  using V = RowVec<T, 1>;
  const int64_t n = B * C;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t b = i / C, c = i - b * C;
    V vz, vx, vh;
    float z, xv, a, rest, u;
    vz.load(gate + b * ldg + c);
    vx.load(x + b * ldx + c);
    vz.get(&z);
    vx.get(&xv);
    gate_of<FORM>(z, xv, a, rest, u);
    const float hn = fmaf(a, state[b * lds + c], u);
    state[b * lds + c] = hn;
    vh.set(&hn);
    vh.store(h + i);
  }
}

// Blocks of a cluster: enough for two blocks per SM, no more than the steps fill.
int cluster_size(int64_t blocks, int64_t T, int64_t steps_per_block) {
  const int64_t want = 2 * (int64_t)num_sms();
  int S = 1;
  while (S < GS_MAX_CLUSTER && blocks * S < want && T > S * steps_per_block) S *= 2;
  return S;
}

template <typename K, typename A>
int launch_clustered(K kernel, const A& args, int threads, int64_t B, int64_t tiles, int S,
                     cudaStream_t stream) {
  if (B * tiles > INT32_MAX / GS_MAX_CLUSTER) return TP_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * tiles * S));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = S;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args, S, tiles));
}

// two bf16 channels per lane: even channels at even strides, 4-byte aligned
bool pairs_ok(const GatedScanArgs& a) {
  auto al = [](const void* p) { return (((uintptr_t)p) & 3) == 0; };
  return a.dtype == TP_DTYPE_BF16 && a.C % 2 == 0 && a.gate_sb % 2 == 0 && a.gate_st % 2 == 0 &&
         a.x_sb % 2 == 0 && a.x_st % 2 == 0 && al(a.gate) && al(a.x) &&
         (a.h == nullptr || al(a.h));
}

template <typename T, int CPL, int FORM>
int fwd(const GatedScanArgs& a, cudaStream_t stream) {
  constexpr int L = 16, W = 8;
  const int64_t tiles = ceil_div(a.C, (int64_t)(32 * CPL));
  const int S = cluster_size(a.B * tiles, a.T, L * W);
  return launch_clustered(gated_scan_fwd_kernel<T, CPL, FORM, L, W>, a, 32 * W, a.B, tiles, S,
                          stream);
}

template <typename T, int CPL, int FORM>
int bwd(const GatedScanBwdArgs& g, cudaStream_t stream) {
  constexpr int L = 8, W = 8;
  const int64_t tiles = ceil_div(g.f.C, (int64_t)(32 * CPL));
  const int S = cluster_size(g.f.B * tiles, g.f.T, L * W);
  return launch_clustered(gated_scan_bwd_kernel<T, CPL, FORM, L, W>, g, 32 * W, g.f.B, tiles, S,
                          stream);
}

}  // namespace

int launch_gated_scan_fwd(const GatedScanArgs& a, cudaStream_t stream) {
  const bool sig = a.form == TP_GATE_SIGMOID;
  if (a.dtype == TP_DTYPE_F32)
    return sig ? fwd<float, 1, TP_GATE_SIGMOID>(a, stream)
               : fwd<float, 1, TP_GATE_DECAY>(a, stream);
  if (pairs_ok(a))
    return sig ? fwd<bf16_t, 2, TP_GATE_SIGMOID>(a, stream)
               : fwd<bf16_t, 2, TP_GATE_DECAY>(a, stream);
  return sig ? fwd<bf16_t, 1, TP_GATE_SIGMOID>(a, stream)
             : fwd<bf16_t, 1, TP_GATE_DECAY>(a, stream);
}

int launch_gated_scan_bwd(const GatedScanBwdArgs& g, cudaStream_t stream) {
  const bool sig = g.f.form == TP_GATE_SIGMOID;
  if (g.f.dtype == TP_DTYPE_F32)
    return sig ? bwd<float, 1, TP_GATE_SIGMOID>(g, stream)
               : bwd<float, 1, TP_GATE_DECAY>(g, stream);
  auto al = [](const void* p) { return (((uintptr_t)p) & 3) == 0; };
  if (pairs_ok(g.f) && al(g.dh) && al(g.dgate) && al(g.dx))
    return sig ? bwd<bf16_t, 2, TP_GATE_SIGMOID>(g, stream)
               : bwd<bf16_t, 2, TP_GATE_DECAY>(g, stream);
  return sig ? bwd<bf16_t, 1, TP_GATE_SIGMOID>(g, stream)
             : bwd<bf16_t, 1, TP_GATE_DECAY>(g, stream);
}

int launch_gated_scan_step(int dtype, int form, int64_t B, int64_t C, const void* gate,
                           int64_t ldg, const void* x, int64_t ldx, float* state, int64_t lds,
                           void* h, cudaStream_t stream) {
  const int64_t want = ceil_div(B * C, (int64_t)256), cap = (int64_t)num_sms() * 16;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  const bool sig = form == TP_GATE_SIGMOID;
#define GS_STEP(T, F)                                                                      \
  gated_scan_step_kernel<T, F><<<grid, 256, 0, stream>>>(B, C, (const T*)gate, ldg,        \
                                                         (const T*)x, ldx, state, lds, (T*)h)
  if (dtype == TP_DTYPE_F32) {
    if (sig) GS_STEP(float, TP_GATE_SIGMOID);
    else GS_STEP(float, TP_GATE_DECAY);
  } else {
    if (sig) GS_STEP(bf16_t, TP_GATE_SIGMOID);
    else GS_STEP(bf16_t, TP_GATE_DECAY);
  }
#undef GS_STEP
  return launch_status();
}

}  // namespace tp
