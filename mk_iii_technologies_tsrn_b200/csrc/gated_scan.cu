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
// (two per lane where the layout allows: 128 or 256 bytes a row, and packed
// fp32 pairs in the arithmetic) and L consecutive steps; the W warps of a block
// own consecutive runs, and the S blocks of a thread-block cluster consecutive
// groups of those.  An iteration of S * W * L steps forms every warp's (A, H),
// exchanges them through shared memory (between the cluster's blocks through
// distributed shared memory, one cluster barrier), applies the runs in order to
// the carried state, and runs each warp's steps again from its own starting
// state.  So the inputs are read once, the order of every operation is fixed
// (the same bits on each call), and few channels still spread over many SMs.
// The inputs of the next iterations are on their way meanwhile: each thread
// copies its own elements asynchronously into shared memory, one or two
// iterations ahead, and reads only those, so the copies need no barrier.
//
// The backward walks the iterations from the end with the mirrored recurrence
//   g_t = dh_t + c_{t+1},  c_t = a_t g_t   (c_t: gradient of h_{t-1})
// and forms da_t = g_t h_{t-1} from states it recomputes in fp32: the forward
// keeps one state per 64 steps.  It reads gate, x and dh once and writes dgate
// and dx: like the forward it is bound by memory.
#include <initializer_list>

#include "maxplus_internal.cuh"
#include "rowvec.cuh"

namespace tp {

namespace {

#ifndef GS_MINB
#define GS_MINB 2
#endif
#ifndef GS_WANT
#define GS_WANT 1.0
#endif
constexpr int GS_MAX_CLUSTER = 16;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One or two channels of a lane.
template <int CPL>
struct Lane;
template <>
struct Lane<1> {
  float v;
  __device__ __forceinline__ static Lane all(float f) { return {f}; }
  __device__ __forceinline__ float at(int) const { return v; }
  __device__ __forceinline__ void put(int, float f) { v = f; }
};
template <>
struct Lane<2> {
  float2 v;
  __device__ __forceinline__ static Lane all(float f) { return {make_float2(f, f)}; }
  __device__ __forceinline__ float at(int k) const { return k ? v.y : v.x; }
  __device__ __forceinline__ void put(int k, float f) { (k ? v.y : v.x) = f; }
};
// (rounded one by one: the compiler may not join a product and a sum into one
// rounding for one channel per lane and not for two)
__device__ __forceinline__ Lane<1> fma_(Lane<1> a, Lane<1> b, Lane<1> c) {
  return {fmaf(a.v, b.v, c.v)};
}
__device__ __forceinline__ Lane<2> fma_(Lane<2> a, Lane<2> b, Lane<2> c) {
  return {tp_fma2(a.v, b.v, c.v)};
}
__device__ __forceinline__ Lane<1> mul_(Lane<1> a, Lane<1> b) { return {__fmul_rn(a.v, b.v)}; }
__device__ __forceinline__ Lane<2> mul_(Lane<2> a, Lane<2> b) { return {tp_mul2(a.v, b.v)}; }
__device__ __forceinline__ Lane<1> add_(Lane<1> a, Lane<1> b) { return {__fadd_rn(a.v, b.v)}; }
__device__ __forceinline__ Lane<2> add_(Lane<2> a, Lane<2> b) { return {tp_add2(a.v, b.v)}; }

// The run (A, H) of a block, sent into the same shared-memory place of the
// cluster's block `rank`; the bytes count on that block's barrier, so the
// receiver needs no fence, and the sender does not wait for its global stores
// as a cluster barrier's release would.
template <int CPL>
struct __align__(8 * CPL) Run {
  Lane<CPL> a, h;
};
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(r)
               : "r"(tp_smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void send_run(Run<1>* to, uint64_t* bar, uint32_t rank, Run<1> r) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::
          "r"(at_rank(to, rank)), "f"(r.a.v), "f"(r.h.v), "r"(at_rank(bar, rank))
      : "memory");
}
__device__ __forceinline__ void send_run(Run<2>* to, uint64_t* bar, uint32_t rank, Run<2> r) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 "
      "[%0], {%1, %2, %3, %4}, [%5];" ::"r"(at_rank(to, rank)),
      "f"(r.a.v.x), "f"(r.a.v.y), "f"(r.h.v.x), "f"(r.h.v.y), "r"(at_rank(bar, rank))
      : "memory");
}

// CPL channels in storage, as one word of shared memory or a register
template <typename T, int CPL>
__device__ __forceinline__ Lane<CPL> unpack(const RowVec<T, CPL>& r) {
  float f[CPL];
  r.get(f);
  Lane<CPL> l;
#pragma unroll
  for (int k = 0; k < CPL; ++k) l.put(k, f[k]);
  return l;
}
template <typename T, int CPL>
__device__ __forceinline__ void store_lane(T* p, Lane<CPL> l) {
  float f[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k) f[k] = l.at(k);
  RowVec<T, CPL> r;
  r.set(f);
  r.store_stream(p);
}

// Copies of a warp's n <= L rows of 32 CPL channels into shared memory
// [L][32] of V.  WIDE: 16 bytes per lane, several rows per instruction (all rows
// 16-byte aligned); else every lane its own channels, asynchronously where they
// make at least four bytes.  The caller synchronises the warp around them.
template <typename T, int CPL, int L, bool WIDE>
struct Rows {
  static constexpr int PER = 32 * CPL * (int)sizeof(T) / 16;   // 16-byte pieces of a row
  // the element of the row at which this lane's copies begin
  __device__ __forceinline__ static int first_channel(int lane) {
    return WIDE ? (lane % PER) * (16 / (int)sizeof(T)) : lane * CPL;
  }
  // p: this lane's element of the first row
  __device__ __forceinline__ static void copy(RowVec<T, CPL>* s, const T* p, int64_t stride,
                                              int n, int lane) {
    if constexpr (WIDE) {
      constexpr int ROWS = 32 / PER;      // rows per instruction
      char* d = reinterpret_cast<char*>(s) + lane * 16;
      const int r = lane / PER;
      p += r * stride;
#pragma unroll
      for (int i = 0; i < L; i += ROWS) {
        if (i + r < n)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tp_smem_addr(d + i * PER * 16)),
                       "l"(p)
                       : "memory");
        p += ROWS * stride;
      }
    } else {
      s += lane;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        if (i < n) {
          if constexpr (sizeof(T) * CPL == 8)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(tp_smem_addr(s + i * 32)),
                         "l"(p)
                         : "memory");
          else if constexpr (sizeof(T) * CPL == 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tp_smem_addr(s + i * 32)),
                         "l"(p)
                         : "memory");
          else
            s[i * 32].load_stream(p);
        }
        p += stride;
      }
    }
  }
};

// A product of gates kept finite: gates above 1 may overflow it, and a zero
// state must stay zero.  (A NaN gate is NaN in the run's result as well.)
template <int CPL>
__device__ __forceinline__ Lane<CPL> finite(Lane<CPL> a) {
#pragma unroll
  for (int k = 0; k < CPL; ++k)
    a.put(k, fminf(fmaxf(a.at(k), -3.402823466e38f), 3.402823466e38f));
  return a;
}

// Gate as the recurrence's a, and 1 - a in the sigmoid form.  bf16 storage: the
// gate comes from 2^x with the argument rounded once, relative error about
// (8 + 1.5 |z|) 2^-24, far below the 2^-9 of the stored result; fp32: to fp32
// accuracy.
template <typename T, int FORM>
__device__ __forceinline__ void gate_of(float z, float& a, float& rest) {
  if constexpr (FORM == TP_GATE_SIGMOID) {
    if constexpr (sizeof(T) == 2) fast_sigmoid_pair(z, a, rest);
    else sigmoid_pair(z, a, rest);
  } else {
    a = z;
    rest = 1.0f;
  }
}
template <typename T, int FORM, int CPL>
__device__ __forceinline__ void gates_of(Lane<CPL> z, Lane<CPL>& a, Lane<CPL>& rest) {
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    float p, q;
    gate_of<T, FORM>(z.at(k), p, q);
    a.put(k, p);
    rest.put(k, q);
  }
}

template <typename T, int CPL>
struct Place {
  int64_t b, c;       // batch row, this lane's first channel
  bool in;            // the lane has channels
  int64_t len;        // live steps of the row
  int rank;           // block of the cluster
  __device__ __forceinline__ Place(const GatedScanArgs& a, int S, int64_t tiles) {
    const int64_t id = blockIdx.x / S;
    rank = S > 1 ? (int)cluster_rank() : 0;
    b = id / tiles;
    c = (id - b * tiles) * (32 * CPL) + (threadIdx.x & 31) * CPL;
    in = c < a.C;
    len = a.T;
    if (a.lengths) {
      const int64_t n = a.lengths[b];
      len = n < 0 ? 0 : (n < a.T ? n : a.T);
    }
  }
  __device__ __forceinline__ Lane<CPL> load(const float* p, int64_t row, int64_t C) const {
    Lane<CPL> l = Lane<CPL>::all(0.0f);
    if (p != nullptr && in) {
#pragma unroll
      for (int k = 0; k < CPL; ++k) l.put(k, p[row * C + c + k]);
    }
    return l;
  }
  __device__ __forceinline__ void store(float* p, int64_t row, int64_t C, Lane<CPL> l) const {
    if (p != nullptr && in) {
#pragma unroll
      for (int k = 0; k < CPL; ++k) p[row * C + c + k] = l.at(k);
    }
  }
};

// steps of [t0, t0 + L) below `end`
template <int L>
__device__ __forceinline__ int steps_below(int64_t end, int64_t t0) {
  const int64_t n = end - t0;
  return n <= 0 ? 0 : (n < L ? (int)n : L);
}

template <typename T, int CPL, int FORM, int L, int W, int STAGES, bool WIDE>
__global__ void __launch_bounds__(32 * W, GS_MINB)
    gated_scan_fwd_kernel(const GatedScanArgs a, const int S, const int64_t tiles, int* err) {
  using V = RowVec<T, CPL>;
  using N = Lane<CPL>;
  extern __shared__ __align__(16) unsigned char s_raw[];   // [STAGES][2][W][L][32] of V
  __shared__ N s_a[2][W][32], s_h[2][W][32];               // runs of the warps
  V* const raw = reinterpret_cast<V*>(s_raw);
  // runs of the cluster's blocks: [2][S][32], filled by the blocks themselves
  Run<CPL>* const s_blk = reinterpret_cast<Run<CPL>*>(raw + STAGES * 2 * L * 32 * W);
  __shared__ uint64_t s_bar[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place<T, CPL> w(a, S, tiles);
  T* const hp = (T*)a.h + (w.b * a.T) * a.C + w.c;
  const int64_t chunks = ceil_div(a.T, (int64_t)GATED_SCAN_CHUNK);
  const int64_t step = (int64_t)S * W * L;
  const int64_t iters = ceil_div(a.T, step);
  const int64_t mine0 = ((int64_t)w.rank * W + warp) * L;
  N carry = w.load(a.h0, w.b, a.C);

  using R = Rows<T, CPL, L, WIDE>;
  const int64_t c0 = w.c - lane * CPL + R::first_channel(lane);   // this lane copies from here
  const T* const gf = (const T*)a.gate + w.b * a.gate_sb + c0;
  const T* const xf = (const T*)a.x + w.b * a.x_sb + c0;
  const bool copies = c0 < a.C;
  auto fetch = [&](int64_t it) {
    if (it < iters && copies) {
      const int64_t t0 = it * step + mine0;
      const int n = steps_below<L>(w.len, t0);
      V* s = raw + ((it % STAGES) * (2 * W) + warp) * (L * 32);
      R::copy(s, gf + t0 * a.gate_st, a.gate_st, n, lane);
      R::copy(s + W * L * 32, xf + t0 * a.x_st, a.x_st, n, lane);
    }
    tp_cp_async_commit();
  };
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch(k);
  if (S > 1) {     // every block of the cluster has its barriers before the first run is sent
    if (threadIdx.x == 0) {
      tp_mbar_init(&s_bar[0], 1);
      tp_mbar_init(&s_bar[1], 1);
      tp_fence_mbar_init();
    }
    cluster_arrive();
    cluster_wait();
  }
  bool ok = true;
  for (int64_t it = 0; it < iters; ++it) {
    __syncwarp();          // the warp has read the stage that is filled now
    fetch(it + STAGES - 1);
    const int par = (int)(it & 1);
    const int64_t t0 = it * step + mine0;
    const int n = steps_below<L>(w.len, t0);
    tp_cp_async_wait<STAGES - 1>();
    __syncwarp();          // and every lane's copies of this stage are there
    const V* s = raw + ((it % STAGES) * (2 * W) + warp) * (L * 32) + lane;
    N A[L], U[L];
    N pa = N::all(1.0f), ph = N::all(0.0f);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      N rest;
      gates_of<T, FORM>(unpack<T, CPL>(s[i * 32]), A[i], rest);
      U[i] = unpack<T, CPL>(s[(W * L + i) * 32]);
      if constexpr (FORM == TP_GATE_SIGMOID) U[i] = mul_(rest, U[i]);
    }
    if (n < L) {          // past the end the state stays
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (i >= n) {
          A[i] = N::all(1.0f);
          U[i] = N::all(0.0f);
        }
    }
#pragma unroll
    for (int i = 0; i < L; ++i) {
      ph = fma_(A[i], ph, U[i]);
      pa = mul_(pa, A[i]);
    }
    s_a[par][warp][lane] = finite(pa);
    s_h[par][warp][lane] = ph;
    __syncthreads();
    N mine;
    if (S == 1) {
      N h = carry;
      mine = h;
#pragma unroll
      for (int q = 0; q < W; ++q) {
        if (q == warp) mine = h;
        h = fma_(s_a[par][q][lane], h, s_h[par][q][lane]);
      }
      carry = h;
    } else {
      // the runs before this warp's, composed; the last warp has the block's
      N qa = N::all(1.0f), qh = N::all(0.0f);
#pragma unroll
      for (int q = 0; q < W; ++q) {
        if (q < warp || warp == W - 1) {
          const N na = s_a[par][q][lane];
          if (q == warp) {
            mine = qh;     // (last warp: keep the composition up to itself)
            pa = qa;
          }
          qh = fma_(na, qh, s_h[par][q][lane]);
          qa = mul_(qa, na);
        }
      }
      if (warp == W - 1) {
        const Run<CPL> r = {finite(qa), qh};
        for (int q = 0; q < S; ++q)
          send_run(s_blk + (par * S + w.rank) * 32 + lane, &s_bar[par], q, r);
        if (lane == 0) tp_mbar_arrive_expect_tx(&s_bar[par], S * 32 * (int)sizeof(Run<CPL>));
        qa = pa;
        qh = mine;
      }
      // (a wait that runs out is recorded; the blocks stay in step and finish)
      ok = ok && tp_mbar_wait(&s_bar[par], (unsigned)(it >> 1) & 1u, err);
      N h = carry, start = carry;
      for (int q = 0; q < S; ++q) {
        if (q == w.rank) start = h;
        const Run<CPL> r = s_blk[(par * S + q) * 32 + lane];
        h = fma_(r.a, h, r.h);
      }
      carry = h;
      mine = fma_(finite(qa), start, qh);
    }
    if (a.states && t0 < a.T && (t0 % GATED_SCAN_CHUNK) == 0)
      w.store(a.states, w.b * chunks + t0 / GATED_SCAN_CHUNK, a.C, mine);
    T* o = hp + t0 * a.C;
    const int m = steps_below<L>(a.T, t0);
    if (n == L) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        mine = fma_(A[i], mine, U[i]);
        if (w.in) store_lane<T, CPL>(o, mine);
        o += a.C;
      }
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        mine = fma_(A[i], mine, U[i]);
        if (w.in && i < m) store_lane<T, CPL>(o, i < n ? mine : N::all(0.0f));
        o += a.C;
      }
    }
  }
  if (w.rank == 0 && warp == 0) w.store(a.h_last, w.b, a.C, carry);
  if (S > 1) {     // no block leaves while another may still send to it
    cluster_arrive();
    cluster_wait();
  }
}

template <typename T, int CPL, int FORM, int L, int W, int STAGES, bool WIDE>
__global__ void __launch_bounds__(32 * W, GS_MINB)
    gated_scan_bwd_kernel(const GatedScanBwdArgs g, const int S, const int64_t tiles, int* err) {
  static_assert(GATED_SCAN_CHUNK % L == 0 && (W * L) % GATED_SCAN_CHUNK == 0, "");
  using V = RowVec<T, CPL>;
  using N = Lane<CPL>;
  const GatedScanArgs& a = g.f;
  extern __shared__ __align__(16) unsigned char s_raw[];   // [STAGES][3][W][L][32] of V
  __shared__ N s_a[2][W][32], s_h[2][W][32], s_c[2][W][32];   // runs, forwards and backwards
  V* const raw = reinterpret_cast<V*>(s_raw);
  Run<CPL>* const s_blk = reinterpret_cast<Run<CPL>*>(raw + STAGES * 3 * L * 32 * W);
  __shared__ uint64_t s_bar[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place<T, CPL> w(a, S, tiles);
  T* const dgp = (T*)g.dgate + (w.b * a.T) * a.C + w.c;
  T* const dxp = (T*)g.dx + (w.b * a.T) * a.C + w.c;
  const int64_t chunks = ceil_div(a.T, (int64_t)GATED_SCAN_CHUNK);
  const int64_t step = (int64_t)S * W * L;
  const int64_t iters = ceil_div(a.T, step);
  const int64_t mine0 = ((int64_t)w.rank * W + warp) * L;
  // the first warp of this warp's 64-step chunk, whose starting state is kept
  constexpr int WPC = GATED_SCAN_CHUNK / L;
  const int lead = warp - warp % WPC;
  N carry = w.load(g.dh_last, w.b, a.C);

  using R = Rows<T, CPL, L, WIDE>;
  const int64_t c0 = w.c - lane * CPL + R::first_channel(lane);
  const T* const gf = (const T*)a.gate + w.b * a.gate_sb + c0;
  const T* const xf = (const T*)a.x + w.b * a.x_sb + c0;
  const T* const df = (const T*)g.dh + w.b * a.T * a.C + c0;
  const bool copies = c0 < a.C, has_dh = g.dh != nullptr;
  auto fetch = [&](int64_t it) {       // it counts from the end
    if (it < iters && copies) {
      const int64_t t0 = (iters - 1 - it) * step + mine0;
      const int n = steps_below<L>(w.len, t0);
      V* s = raw + ((it % STAGES) * (3 * W) + warp) * (L * 32);
      R::copy(s, gf + t0 * a.gate_st, a.gate_st, n, lane);
      R::copy(s + W * L * 32, xf + t0 * a.x_st, a.x_st, n, lane);
      if (has_dh) R::copy(s + 2 * W * L * 32, df + t0 * a.C, a.C, n, lane);
    }
    tp_cp_async_commit();
  };
  auto first_state = [&](int64_t it) {
    const int64_t t0 = (iters - 1 - it) * step + mine0;
    if (it >= iters || t0 >= w.len) return N::all(0.0f);
    return w.load(a.states, w.b * chunks + t0 / GATED_SCAN_CHUNK, a.C);
  };
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch(k);
  N next = first_state(0);
  if (S > 1) {     // every block of the cluster has its barriers before the first run is sent
    if (threadIdx.x == 0) {
      tp_mbar_init(&s_bar[0], 1);
      tp_mbar_init(&s_bar[1], 1);
      tp_fence_mbar_init();
    }
    cluster_arrive();
    cluster_wait();
  }
  bool ok = true;
  for (int64_t it = 0; it < iters; ++it) {
    __syncwarp();
    fetch(it + STAGES - 1);
    const N first = next;
    next = first_state(it + 1);
    const int par = (int)(it & 1);
    const int64_t t0 = (iters - 1 - it) * step + mine0;
    const int n = steps_below<L>(w.len, t0);
    tp_cp_async_wait<STAGES - 1>();
    __syncwarp();
    const V* s = raw + ((it % STAGES) * (3 * W) + warp) * (L * 32) + lane;
    N A[L], O[L], U[L];      // gate, its complement, input
    N pa = N::all(1.0f), ph = N::all(0.0f);
    auto dh_at = [&](int i) {
      return (has_dh && i < n) ? unpack<T, CPL>(s[(2 * W * L + i) * 32]) : N::all(0.0f);
    };
#pragma unroll
    for (int i = 0; i < L; ++i) {
      gates_of<T, FORM>(unpack<T, CPL>(s[i * 32]), A[i], O[i]);
      U[i] = unpack<T, CPL>(s[(W * L + i) * 32]);
      if constexpr (FORM == TP_GATE_SIGMOID) U[i] = mul_(O[i], U[i]);
    }
    if (n < L) {
#pragma unroll
      for (int i = 0; i < L; ++i)
        if (i >= n) {
          A[i] = N::all(1.0f);
          U[i] = N::all(0.0f);
        }
    }
#pragma unroll
    for (int i = 0; i < L; ++i) {
      ph = fma_(A[i], ph, U[i]);
      pa = mul_(pa, A[i]);
    }
    N gr = dh_at(L - 1);      // g of the run alone
#pragma unroll
    for (int i = L - 2; i >= 0; --i) gr = fma_(A[i + 1], gr, dh_at(i));
    s_a[par][warp][lane] = finite(pa);
    s_h[par][warp][lane] = ph;
    s_c[par][warp][lane] = mul_(A[0], gr);
    __syncthreads();
    N mine;
    if (S == 1) {
      N c = carry;
      mine = c;
#pragma unroll
      for (int q = W - 1; q >= 0; --q) {
        if (q == warp) mine = c;
        c = fma_(s_a[par][q][lane], c, s_c[par][q][lane]);
      }
      carry = c;
    } else {
      // the runs after this warp's, composed; the first warp has the block's
      N qa = N::all(1.0f), qc = N::all(0.0f);
#pragma unroll
      for (int q = W - 1; q >= 0; --q) {
        if (q > warp || warp == 0) {
          const N na = s_a[par][q][lane];
          if (q == warp) {
            mine = qc;
            pa = qa;
          }
          qc = fma_(na, qc, s_c[par][q][lane]);
          qa = mul_(qa, na);
        }
      }
      if (warp == 0) {
        const Run<CPL> r = {finite(qa), qc};
        for (int q = 0; q < S; ++q)
          send_run(s_blk + (par * S + w.rank) * 32 + lane, &s_bar[par], q, r);
        if (lane == 0) tp_mbar_arrive_expect_tx(&s_bar[par], S * 32 * (int)sizeof(Run<CPL>));
        qa = pa;
        qc = mine;
      }
      ok = ok && tp_mbar_wait(&s_bar[par], (unsigned)(it >> 1) & 1u, err);
      N c = carry, start = carry;
      for (int q = S - 1; q >= 0; --q) {
        if (q == w.rank) start = c;
        const Run<CPL> r = s_blk[(par * S + q) * 32 + lane];
        c = fma_(r.a, c, r.h);
      }
      carry = c;
      mine = fma_(finite(qa), start, qc);
    }
    N before[L];      // h_{t-1}
    {
      N h = first;
      for (int q = lead; q < warp; ++q) h = fma_(s_a[par][q][lane], h, s_h[par][q][lane]);
#pragma unroll
      for (int i = 0; i < L; ++i) {
        before[i] = h;
        h = fma_(A[i], h, U[i]);
      }
    }
    T* oz = dgp + (t0 + L - 1) * a.C;
    T* ox = dxp + (t0 + L - 1) * a.C;
    const int m = steps_below<L>(a.T, t0);
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      gr = i == L - 1 ? add_(dh_at(i), mine) : fma_(A[i + 1 < L ? i + 1 : i], gr, dh_at(i));
      N z, x;
      if constexpr (FORM == TP_GATE_SIGMOID) {
        // d(f h + (1 - f) x)/dz = f (1 - f) (h - x) = f ((1 - f) h - u)
        z = mul_(mul_(A[i], gr), fma_(O[i], before[i], mul_(N::all(-1.0f), U[i])));
        x = mul_(gr, O[i]);
      } else {
        z = mul_(gr, before[i]);
        x = gr;
      }
      if (w.in && i < m) {
        store_lane<T, CPL>(oz, i < n ? z : N::all(0.0f));
        store_lane<T, CPL>(ox, i < n ? x : N::all(0.0f));
      }
      oz -= a.C;
      ox -= a.C;
    }
  }
  if (w.rank == 0 && warp == 0) w.store(g.dh0, w.b, a.C, carry);
  if (S > 1) {     // no block leaves while another may still send to it
    cluster_arrive();
    cluster_wait();
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
    gate_of<T, FORM>(z, a, rest);
    u = FORM == TP_GATE_SIGMOID ? rest * xv : xv;
    const float hn = fmaf(a, state[b * lds + c], u);
    state[b * lds + c] = hn;
    vh.set(&hn);
    vh.store(h + i);
  }
}

// Blocks of a cluster: enough for two blocks per SM, no more than the steps
// fill.  It goes by the sizes alone, as L does by the type, so that the order of
// operations, and with it the bits, do not depend on strides and alignment.
int cluster_size(int64_t B, int64_t T, int64_t C, int64_t steps_per_block) {
  const int64_t want = (int64_t)(GS_WANT * num_sms()), blocks = B * ceil_div(C, (int64_t)64);
  int S = 1;
  while (S < GS_MAX_CLUSTER && blocks * S < want && T > S * steps_per_block) S *= 2;
  return S;
}

template <typename K, typename A>
int launch_clustered(K kernel, const A& args, int threads, size_t smem, size_t runs_bytes,
                     int64_t B, int64_t tiles, int S, cudaStream_t stream) {
  if (B * tiles > INT32_MAX / GS_MAX_CLUSTER) return TP_ERR_TOO_LARGE;
  if (S > 1) smem += (size_t)2 * S * runs_bytes;
  cudaError_t e = cudaFuncSetAttribute((const void*)kernel,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess && S > 8)
    e = cudaFuncSetAttribute((const void*)kernel,
                             cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return cuda_status(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * tiles * S));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = S;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 1 : 0;
  int* err = device_error_ptr();
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args, S, tiles, err));
}

// Whether rows, strides and bases are multiples of `bytes`.
bool rows_at(const GatedScanArgs& a, std::initializer_list<const void*> more, int bytes) {
  const uintptr_t m = bytes - 1;
  for (const void* p : {a.gate, a.x})
    if (((uintptr_t)p) & m) return false;
  for (const void* p : more)
    if (((uintptr_t)p) & m) return false;
  const int64_t n = bytes / (a.dtype == TP_DTYPE_F32 ? 4 : 2);
  return a.C % n == 0 && a.gate_sb % n == 0 && a.gate_st % n == 0 && a.x_sb % n == 0 &&
         a.x_st % n == 0;
}

template <typename T, int CPL, int FORM, bool WIDE>
int fwd(const GatedScanArgs& a, cudaStream_t stream) {
#ifdef GS_FL
  constexpr int L = GS_FL, W = GS_FW, STAGES = GS_FS;
#else
  constexpr int L = sizeof(T) == 4 ? 8 : 16, W = 8, STAGES = 3;
#endif
  const int64_t tiles = ceil_div(a.C, (int64_t)(32 * CPL));
  const int S = cluster_size(a.B, a.T, a.C, L * W);
  return launch_clustered(gated_scan_fwd_kernel<T, CPL, FORM, L, W, STAGES, WIDE>, a, 32 * W,
                          (size_t)STAGES * 2 * L * 32 * W * CPL * sizeof(T),
                          32 * sizeof(Run<CPL>), a.B, tiles, S, stream);
}

template <typename T, int CPL, int FORM, bool WIDE>
int bwd(const GatedScanBwdArgs& g, cudaStream_t stream) {
#ifdef GS_BL
  constexpr int L = GS_BL, W = GS_BW, STAGES = GS_BS;
#else
  constexpr int L = 8, W = 8, STAGES = sizeof(T) * CPL == 8 ? 2 : 3;
#endif
  const int64_t tiles = ceil_div(g.f.C, (int64_t)(32 * CPL));
  const int S = cluster_size(g.f.B, g.f.T, g.f.C, L * W);
  return launch_clustered(gated_scan_bwd_kernel<T, CPL, FORM, L, W, STAGES, WIDE>, g, 32 * W,
                          (size_t)STAGES * 3 * L * 32 * W * CPL * sizeof(T),
                          32 * sizeof(Run<CPL>), g.f.B, tiles, S, stream);
}

// Two channels per lane and 16-byte copies where rows are 16-byte aligned, else
// one channel per lane.
template <typename T, int FORM>
int fwd_any(const GatedScanArgs& a, cudaStream_t stream) {
  if (rows_at(a, {a.h}, 16)) return fwd<T, 2, FORM, true>(a, stream);
  return fwd<T, 1, FORM, false>(a, stream);
}
template <typename T, int FORM>
int bwd_any(const GatedScanBwdArgs& g, cudaStream_t stream) {
  if (rows_at(g.f, {g.dh, g.dgate, g.dx}, 16)) return bwd<T, 2, FORM, true>(g, stream);
  return bwd<T, 1, FORM, false>(g, stream);
}

}  // namespace

int launch_gated_scan_fwd(const GatedScanArgs& a, cudaStream_t stream) {
  const bool sig = a.form == TP_GATE_SIGMOID;
  if (a.dtype == TP_DTYPE_F32)
    return sig ? fwd_any<float, TP_GATE_SIGMOID>(a, stream)
               : fwd_any<float, TP_GATE_DECAY>(a, stream);
  return sig ? fwd_any<bf16_t, TP_GATE_SIGMOID>(a, stream)
             : fwd_any<bf16_t, TP_GATE_DECAY>(a, stream);
}

int launch_gated_scan_bwd(const GatedScanBwdArgs& g, cudaStream_t stream) {
  const bool sig = g.f.form == TP_GATE_SIGMOID;
  if (g.f.dtype == TP_DTYPE_F32)
    return sig ? bwd_any<float, TP_GATE_SIGMOID>(g, stream)
               : bwd_any<float, TP_GATE_DECAY>(g, stream);
  return sig ? bwd_any<bf16_t, TP_GATE_SIGMOID>(g, stream)
             : bwd_any<bf16_t, TP_GATE_DECAY>(g, stream);
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
