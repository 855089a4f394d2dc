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
// fp32 pairs in the arithmetic) and L consecutive steps, in registers; the W
// warps of a block own consecutive runs.  An iteration of W * L steps forms every
// warp's (A, H), exchanges them through shared memory, applies the runs in order
// to the carried state, and runs each warp's steps again from its own starting
// state.  So the inputs are read once, the order of every operation is fixed
// (the same bits on each call).  The inputs of the next iterations are on their
// way meanwhile: asynchronous 16-byte copies into shared memory, a warp's own
// rows only, so that they need no block barrier.
//
// Too few rows and channels to fill the GPU that way: time is cut into segments
// with a block each.  A first kernel forms the run of every segment (each warp a
// part of it, nothing to wait for), and the second starts each segment from the
// runs before it, composed in order.  The inputs are then read twice, the second
// time from L2 as far as it holds them.
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
// (The compiler joins a packed product and the packed sum it goes into, and rounds
// them once; single ones written like this it leaves alone.  So that the bits do not
// depend on the channels per lane, no product of mul_ goes into an add_ below.)
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
  // the row and the channel at which this lane's copies begin
  __device__ __forceinline__ static int first_row(int lane) { return WIDE ? lane / PER : 0; }
  __device__ __forceinline__ static int first_channel(int lane) {
    return WIDE ? (lane % PER) * (16 / (int)sizeof(T)) : lane * CPL;
  }
  // p: where this lane's copies begin
  __device__ __forceinline__ static void copy(RowVec<T, CPL>* s, const T* p, int64_t stride,
                                              int n, int lane) {
    if constexpr (WIDE) {
      constexpr int ROWS = 32 / PER;      // rows per instruction
      char* d = reinterpret_cast<char*>(s) + lane * 16;
      n -= lane / PER;
#pragma unroll
      for (int i = 0; i < L; i += ROWS) {
        if (i < n)
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

// Gates above 1 may overflow a run's product, which the recurrence itself need not do:
// its states may be small, or zero, or end at a gate of 0.  A product that met a zero
// gate after its overflow (inf * 0) is 0.  (A NaN gate is NaN in the run's result as
// well, whatever the product.)  One that stays infinite makes the state so, except a
// zero state, which stays what the run's result is.  (Sigmoids are at most 1.)
template <int FORM, int CPL>
__device__ __forceinline__ Lane<CPL> product(Lane<CPL> a) {
  if constexpr (FORM == TP_GATE_DECAY) {
#pragma unroll
    for (int k = 0; k < CPL; ++k) a.put(k, a.at(k) != a.at(k) ? 0.0f : a.at(k));
  }
  return a;
}
// the run of product `a` and result `r` applied to a state
template <int FORM, int CPL>
__device__ __forceinline__ Lane<CPL> apply(Lane<CPL> a, Lane<CPL> state, Lane<CPL> r) {
  if constexpr (FORM == TP_GATE_DECAY) {
#pragma unroll
    for (int k = 0; k < CPL; ++k) a.put(k, state.at(k) == 0.0f ? 0.0f : a.at(k));
  }
  return fma_(a, state, r);
}

// Gate as the recurrence's a, and 1 - a in the sigmoid form.  bf16 storage: from
// 2^x with the argument rounded once, the smaller of the two to a relative
// (8 + 1.5 |z|) 2^-24; fp32: to fp32 accuracy.  Either way the larger one is 1 less
// the smaller, off by half a step and little more: states at the rows' ends, those
// kept for the backward and the gradient of h0 are fp32 sums over many steps, and
// have the error of the recurrence in fp32 with rounded gates, or less.
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
  if constexpr (FORM == TP_GATE_SIGMOID && sizeof(T) == 2 && CPL == 2) {
    fast_sigmoid_pair2(z.v, a.v, rest.v);
  } else {
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      float p, q;
      gate_of<T, FORM>(z.at(k), p, q);
      a.put(k, p);
      rest.put(k, q);
    }
  }
}

template <typename T, int CPL>
struct Place {
  int64_t b, c;       // batch row, this lane's first channel
  bool in;            // the lane has channels
  int64_t len;        // live steps of the row
  int64_t begin, end; // steps of the block's segment
  int seg;
  __device__ __forceinline__ Place(const GatedScanArgs& a, int64_t tiles) {
    const int64_t id = blockIdx.x / a.segs;
    seg = (int)(blockIdx.x - id * a.segs);
    b = id / tiles;
    c = (id - b * tiles) * (32 * CPL) + (threadIdx.x & 31) * CPL;
    in = c < a.C;
    len = a.T;
    if (a.lengths) {
      const int64_t n = a.lengths[b];
      len = n < 0 ? 0 : (n < a.T ? n : a.T);
    }
    begin = seg * a.seg_len;
    end = begin + a.seg_len < a.T ? begin + a.seg_len : a.T;
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

// The run of every segment: runs [B][segs][2][C], products then results.  Each
// of the block's warps takes an eighth of the segment, L steps at a time, with
// the copies of the next steps on their way.  REVERSE: the backward's runs.
template <typename T, int CPL, int FORM, int L, int W, int STAGES, bool WIDE, bool REVERSE>
__global__ void __launch_bounds__(32 * W)
    gated_scan_runs_kernel(const GatedScanArgs a, const T* dh, const int64_t tiles) {
  using V = RowVec<T, CPL>;
  using N = Lane<CPL>;
  using R = Rows<T, CPL, L, WIDE>;
  extern __shared__ __align__(16) unsigned char s_raw[];   // [STAGES][W][2][L][32] of V
  __shared__ N s_a[W][32], s_h[W][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place<T, CPL> w(a, tiles);
  if (w.seg == (REVERSE ? 0 : a.segs - 1)) return;      // nothing follows it
  const int64_t part = a.seg_len / W;                   // a multiple of L
  const int64_t lo = w.begin + warp * part;
  const int64_t hi = min(lo + part, w.len);
  const int batches = hi > lo ? (int)ceil_div(hi - lo, (int64_t)L) : 0;
  const int64_t ost = REVERSE ? a.C : a.x_st;           // the other operand: dh or x
  const bool has = !REVERSE || dh != nullptr;
  const int64_t c0 = w.c - lane * CPL + R::first_channel(lane);
  const int64_t r0 = lo + (REVERSE ? (int64_t)(batches - 1) * L : 0) + R::first_row(lane);
  const T* gf = (const T*)a.gate + w.b * a.gate_sb + r0 * a.gate_st + c0;
  const T* of = (REVERSE ? dh + w.b * a.T * a.C : (const T*)a.x + w.b * a.x_sb) + r0 * ost + c0;
  const int64_t gate_step = (REVERSE ? -L : L) * a.gate_st, o_step = (REVERSE ? -L : L) * ost;
  V* const raw = reinterpret_cast<V*>(s_raw) + warp * (2 * L * 32);
  int next = 0, filling = 0, reading = 0;
  // live steps of batch k: all but those of the last one are full
  auto live = [&](int k) {
    return steps_below<L>(hi, lo + (int64_t)(REVERSE ? batches - 1 - k : k) * L);
  };
  auto fetch = [&]() {
    if (next < batches && c0 < a.C) {
      V* s = raw + filling * (W * 2 * L * 32);
      const int n = live(next);
      R::copy(s, gf, a.gate_st, n, lane);
      if (has) R::copy(s + L * 32, of, ost, n, lane);
    }
    tp_cp_async_commit();
    ++next;
    gf += gate_step;
    of += o_step;
    filling = filling + 1 == STAGES ? 0 : filling + 1;
  };
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch();
  // REVERSE: ph is the g of the last step, of which its gate `ga` makes c
  N pa = N::all(1.0f), ph = N::all(0.0f), ga = N::all(0.0f);
  for (int k = 0; k < batches; ++k) {
    __syncwarp();
    fetch();
    tp_cp_async_wait<STAGES - 1>();
    __syncwarp();
    const V* s = raw + reading * (W * 2 * L * 32) + lane;
    reading = reading + 1 == STAGES ? 0 : reading + 1;
    const int n = live(k);
    auto run = [&](auto all) {
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const int i = REVERSE ? L - 1 - j : j;
        if (all.value || i < n) {
          N A, rest, U = N::all(0.0f);
          gates_of<T, FORM>(unpack<T, CPL>(s[i * 32]), A, rest);
          if (has) U = unpack<T, CPL>(s[(L + i) * 32]);
          if constexpr (REVERSE) {
            ph = fma_(ga, ph, U);
            ga = A;
          } else {
            if constexpr (FORM == TP_GATE_SIGMOID) U = mul_(rest, U);
            ph = fma_(A, ph, U);
          }
          pa = mul_(pa, A);
        }
      }
    };
    if (n == L) run(std::true_type());
    else run(std::false_type());
  }
  s_a[warp][lane] = product<FORM>(pa);
  s_h[warp][lane] = REVERSE ? mul_(ga, ph) : ph;
  __syncthreads();
  if (warp != 0) return;
  pa = N::all(1.0f);
  ph = N::all(0.0f);
#pragma unroll
  for (int k = 0; k < W; ++k) {
    const int q = REVERSE ? W - 1 - k : k;
    ph = apply<FORM>(s_a[q][lane], ph, s_h[q][lane]);
    pa = mul_(pa, s_a[q][lane]);
  }
  const int64_t row = (w.b * a.segs + w.seg) * 2;
  w.store(a.runs, row, a.C, product<FORM>(pa));
  w.store(a.runs, row + 1, a.C, ph);
}

// The state before (REVERSE: the gradient after) the block's segment: the runs of
// the segments before (after) it applied to `carry`.  The warps compose an equal
// share each, through `s_a`, `s_h`, and all apply the shares in order.
template <typename T, int CPL, int FORM, int W, bool REVERSE>
__device__ __forceinline__ Lane<CPL> segment_start(const GatedScanArgs& a, const Place<T, CPL>& w,
                                                   Lane<CPL> carry, Lane<CPL> (*s_a)[32],
                                                   Lane<CPL> (*s_h)[32], int warp, int lane) {
  using N = Lane<CPL>;
  if (a.segs == 1) return carry;
  const int n = REVERSE ? a.segs - 1 - w.seg : w.seg;    // segments to apply
  const int per = (n + W - 1) / W;
  const int lo = min(n, warp * per), hi = min(n, lo + per);
  N pa = N::all(1.0f), ph = N::all(0.0f);
#pragma unroll 4
  for (int k = lo; k < hi; ++k) {
    const int64_t row = (w.b * a.segs + (REVERSE ? a.segs - 1 - k : k)) * 2;
    const N ra = w.load(a.runs, row, a.C), rh = w.load(a.runs, row + 1, a.C);
    ph = apply<FORM>(ra, ph, rh);
    pa = mul_(pa, ra);
  }
  s_a[warp][lane] = product<FORM>(pa);
  s_h[warp][lane] = ph;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < W; ++q) carry = apply<FORM>(s_a[q][lane], carry, s_h[q][lane]);
  return carry;
}

template <typename T, int CPL, int FORM, int L, int W, int STAGES, bool WIDE>
__global__ void __launch_bounds__(32 * W, 2)
    gated_scan_fwd_kernel(const GatedScanArgs a, const int64_t tiles) {
  using V = RowVec<T, CPL>;
  using N = Lane<CPL>;
  extern __shared__ __align__(16) unsigned char s_raw[];   // [STAGES][2][W][L][32] of V
  __shared__ N s_a[2][W][32], s_h[2][W][32];               // runs of the warps
  V* const raw = reinterpret_cast<V*>(s_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place<T, CPL> w(a, tiles);
  T* const hp = (T*)a.h + (w.b * a.T) * a.C + w.c;
  const int64_t chunks = ceil_div(a.T, (int64_t)GATED_SCAN_CHUNK);
  constexpr int step = W * L;
  const int64_t iters = ceil_div(w.end - w.begin, (int64_t)step);
  const int64_t mine0 = w.begin + warp * L;
  N carry = w.load(a.h0, w.b, a.C);

  using R = Rows<T, CPL, L, WIDE>;
  const int64_t c0 = w.c - lane * CPL + R::first_channel(lane);   // this lane copies from here
  const int64_t r0 = mine0 + R::first_row(lane);
  const T* gf = (const T*)a.gate + w.b * a.gate_sb + r0 * a.gate_st + c0;
  const T* xf = (const T*)a.x + w.b * a.x_sb + r0 * a.x_st + c0;
  const int64_t gate_step = step * a.gate_st, x_step = step * a.x_st;
  // live steps of the segment from the next copies on
  int64_t left = c0 < a.C ? min(w.len, w.end) - mine0 : 0;
  int filling = 0, reading = 0;                     // stages
  auto fetch = [&]() {                              // one iteration further each time
    const int n = left <= 0 ? 0 : (left < L ? (int)left : L);
    V* s = raw + (filling * (2 * W) + warp) * (L * 32);
    if (n > 0) {
      R::copy(s, gf, a.gate_st, n, lane);
      R::copy(s + W * L * 32, xf, a.x_st, n, lane);
    }
    tp_cp_async_commit();
    gf += gate_step;
    xf += x_step;
    left -= step;
    filling = filling + 1 == STAGES ? 0 : filling + 1;
  };
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch();
  carry = segment_start<T, CPL, FORM, W, false>(a, w, carry, s_a[1], s_h[1], warp, lane);
  for (int64_t it = 0; it < iters; ++it) {
    __syncwarp();          // the warp has read the stage that is filled now
    fetch();
    const int par = (int)(it & 1);
    const int64_t t0 = mine0 + it * step;
    const int n = steps_below<L>(w.len, t0);
    tp_cp_async_wait<STAGES - 1>();
    __syncwarp();          // and every lane's copies of this stage are there
    const V* s = raw + (reading * (2 * W) + warp) * (L * 32) + lane;
    reading = reading + 1 == STAGES ? 0 : reading + 1;
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
    s_a[par][warp][lane] = product<FORM>(pa);
    s_h[par][warp][lane] = ph;
    __syncthreads();
    N mine = carry, h = carry;
#pragma unroll
    for (int q = 0; q < W; ++q) {
      if (q == warp) mine = h;
      h = apply<FORM>(s_a[par][q][lane], h, s_h[par][q][lane]);
    }
    carry = h;
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
  if (w.seg == a.segs - 1 && warp == 0) w.store(a.h_last, w.b, a.C, carry);
}

template <typename T, int CPL, int FORM, int L, int W, int STAGES, bool WIDE>
__global__ void __launch_bounds__(32 * W, 2)
    gated_scan_bwd_kernel(const GatedScanBwdArgs g, const int64_t tiles) {
  static_assert(GATED_SCAN_CHUNK % L == 0 && (W * L) % GATED_SCAN_CHUNK == 0, "");
  using V = RowVec<T, CPL>;
  using N = Lane<CPL>;
  const GatedScanArgs& a = g.f;
  extern __shared__ __align__(16) unsigned char s_raw[];   // [STAGES][3][W][L][32] of V
  __shared__ N s_a[2][W][32], s_h[2][W][32], s_c[2][W][32];   // runs, forwards and backwards
  V* const raw = reinterpret_cast<V*>(s_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place<T, CPL> w(a, tiles);
  T* const dgp = (T*)g.dgate + (w.b * a.T) * a.C + w.c;
  T* const dxp = (T*)g.dx + (w.b * a.T) * a.C + w.c;
  const int64_t chunks = ceil_div(a.T, (int64_t)GATED_SCAN_CHUNK);
  constexpr int step = W * L;
  const int64_t iters = ceil_div(w.end - w.begin, (int64_t)step);
  const int64_t mine0 = w.begin + warp * L;
  // the first warp of this warp's 64-step chunk, whose starting state is kept
  constexpr int WPC = GATED_SCAN_CHUNK / L;
  const int lead = warp - warp % WPC;
  N carry = w.load(g.dh_last, w.b, a.C);

  using R = Rows<T, CPL, L, WIDE>;
  const int64_t c0 = w.c - lane * CPL + R::first_channel(lane);
  const int64_t r0 = (iters - 1) * step + mine0 + R::first_row(lane);
  const T* gf = (const T*)a.gate + w.b * a.gate_sb + r0 * a.gate_st + c0;
  const T* xf = (const T*)a.x + w.b * a.x_sb + r0 * a.x_st + c0;
  const T* df = (const T*)g.dh + (w.b * a.T + r0) * a.C + c0;
  const int64_t gate_step = step * a.gate_st, x_step = step * a.x_st, d_step = step * a.C;
  const bool has_dh = g.dh != nullptr;
  // live steps from the next copies on, and copies left
  int64_t left = w.len - ((iters - 1) * step + mine0), todo = c0 < a.C ? iters : 0;
  int filling = 0, reading = 0;
  auto fetch = [&]() {                 // one iteration towards the start each time
    const int n = left <= 0 ? 0 : (left < L ? (int)left : L);
    V* s = raw + (filling * (3 * W) + warp) * (L * 32);
    if (n > 0 && todo > 0) {
      R::copy(s, gf, a.gate_st, n, lane);
      R::copy(s + W * L * 32, xf, a.x_st, n, lane);
      if (has_dh) R::copy(s + 2 * W * L * 32, df, a.C, n, lane);
    }
    tp_cp_async_commit();
    gf -= gate_step;
    xf -= x_step;
    df -= d_step;
    left += step;
    --todo;
    filling = filling + 1 == STAGES ? 0 : filling + 1;
  };
  auto first_state = [&](int64_t it) {
    const int64_t t0 = (iters - 1 - it) * step + mine0;
    if (it >= iters || t0 >= w.len) return N::all(0.0f);
    return w.load(a.states, w.b * chunks + t0 / GATED_SCAN_CHUNK, a.C);
  };
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch();
  N next = first_state(0);
  carry = segment_start<T, CPL, FORM, W, true>(a, w, carry, s_a[1], s_c[1], warp, lane);
  for (int64_t it = 0; it < iters; ++it) {
    __syncwarp();
    fetch();
    const N first = next;
    next = first_state(it + 1);
    const int par = (int)(it & 1);
    const int64_t t0 = (iters - 1 - it) * step + mine0;
    const int n = steps_below<L>(w.len, t0);
    tp_cp_async_wait<STAGES - 1>();
    __syncwarp();
    const V* s = raw + (reading * (3 * W) + warp) * (L * 32) + lane;
    reading = reading + 1 == STAGES ? 0 : reading + 1;
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
    s_a[par][warp][lane] = product<FORM>(pa);
    s_h[par][warp][lane] = ph;
    s_c[par][warp][lane] = mul_(A[0], gr);
    __syncthreads();
    N mine = carry, c = carry;
#pragma unroll
    for (int q = W - 1; q >= 0; --q) {
      if (q == warp) mine = c;
      c = apply<FORM>(s_a[par][q][lane], c, s_c[par][q][lane]);
    }
    carry = c;
    N before[L];      // h_{t-1}
    {
      N h = first;
      for (int q = lead; q < warp; ++q) h = apply<FORM>(s_a[par][q][lane], h, s_h[par][q][lane]);
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
  if (w.seg == 0 && warp == 0) w.store(g.dh0, w.b, a.C, carry);
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

// Warps of a block, and steps of a warp's run.  More steps per iteration spread
// its fixed costs (exchange, barrier): forward 16 x 4096 x 1024 fp32 with 16
// steps and two stages 131 us, with 8 steps and three stages 156 us.  The
// backward holds twice the registers per step: 8 (16 spill or halve the blocks:
// 232 against 238 us).
constexpr int GS_W = 8;
constexpr int GS_FWD_L = 16, GS_BWD_L = 8, GS_RUN_L = 8;
constexpr int GS_RUN_STAGES = 3;

template <typename K, typename A, typename... More>
int launch_blocks(K kernel, int64_t blocks, size_t smem, cudaStream_t stream, const A& args,
                  More... more) {
  if (smem > 24 * 1024) {      // beside up to 12 KB of the kernels' own
    const int st = allow_smem((const void*)kernel, smem);
    if (st != TP_OK) return st;
  }
  kernel<<<(unsigned)blocks, 32 * GS_W, smem, stream>>>(args, more...);
  return launch_status();
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
  constexpr int L = GS_FWD_L, W = GS_W, STAGES = 2;
  const int64_t tiles = ceil_div(a.C, (int64_t)(32 * CPL));
  const int64_t blocks = a.B * tiles * a.segs;
  if (blocks > INT32_MAX) return TP_ERR_TOO_LARGE;
  if (a.segs > 1) {
    constexpr int RL = GS_RUN_L, RS = GS_RUN_STAGES;
    const int st =
        launch_blocks(gated_scan_runs_kernel<T, CPL, FORM, RL, W, RS, WIDE, false>, blocks,
                      (size_t)RS * 2 * RL * 32 * W * CPL * sizeof(T), stream, a,
                      (const T*)nullptr, tiles);
    if (st != TP_OK) return st;
  }
  return launch_blocks(gated_scan_fwd_kernel<T, CPL, FORM, L, W, STAGES, WIDE>, blocks,
                       (size_t)STAGES * 2 * L * 32 * W * CPL * sizeof(T), stream, a, tiles);
}

template <typename T, int CPL, int FORM, bool WIDE>
int bwd(const GatedScanBwdArgs& g, cudaStream_t stream) {
  constexpr int L = GS_BWD_L, W = GS_W, STAGES = sizeof(T) * CPL == 8 ? 2 : 3;
  const int64_t tiles = ceil_div(g.f.C, (int64_t)(32 * CPL));
  const int64_t blocks = g.f.B * tiles * g.f.segs;
  if (blocks > INT32_MAX) return TP_ERR_TOO_LARGE;
  if (g.f.segs > 1) {
    constexpr int RL = GS_RUN_L, RS = GS_RUN_STAGES;
    const int st = launch_blocks(gated_scan_runs_kernel<T, CPL, FORM, RL, W, RS, WIDE, true>,
                                 blocks, (size_t)RS * 2 * RL * 32 * W * CPL * sizeof(T), stream,
                                 g.f, (const T*)g.dh, tiles);
    if (st != TP_OK) return st;
  }
  return launch_blocks(gated_scan_bwd_kernel<T, CPL, FORM, L, W, STAGES, WIDE>, blocks,
                       (size_t)STAGES * 3 * L * 32 * W * CPL * sizeof(T), stream, g, tiles);
}

// Two channels per lane where rows begin on a pair, with 16-byte copies where they
// begin on 16 bytes, else one channel per lane (16 x 4096 bf16, sigmoid, forward and
// backward: 1024 channels 80 and 166 us, 1020: 110 and 201,
// 1023: 195 and 389 us; the backward of fp32 pairs copied one by one is slower than
// single channels, 16 x 4096 x 1022: 368 against 324 us).
template <typename T, int FORM>
int fwd_any(const GatedScanArgs& a, cudaStream_t stream) {
  if (rows_at(a, {a.h}, 16)) return fwd<T, 2, FORM, true>(a, stream);
  if (rows_at(a, {a.h}, 2 * sizeof(T))) return fwd<T, 2, FORM, false>(a, stream);
  return fwd<T, 1, FORM, false>(a, stream);
}
template <typename T, int FORM>
int bwd_any(const GatedScanBwdArgs& g, cudaStream_t stream) {
  if (rows_at(g.f, {g.dh, g.dgate, g.dx}, 16)) return bwd<T, 2, FORM, true>(g, stream);
  if constexpr (sizeof(T) == 2)
    if (rows_at(g.f, {g.dh, g.dgate, g.dx}, 2 * sizeof(T)))
      return bwd<T, 2, FORM, false>(g, stream);
  return bwd<T, 1, FORM, false>(g, stream);
}

}  // namespace

// Segments of time.  A cut costs a second reading (three arrays forwards become
// five, five backwards become seven), so only rows and channels for less than a
// third of the SMs are cut forwards (4 x 8192 x 1024 fp32, 64 blocks: 95 us in
// one piece, 121 us cut; 2 x 8192 x 1024: 95 and 69 us), less than a half
// backwards (4 x 8192 x 1024: 209 us in one piece, 159 us cut), into about four
// blocks per SM, of at least 256 steps.  The cut goes by the sizes alone, as L
// does by the direction, so that the order of operations, and with it the bits,
// do not depend on strides and alignment.
GatedScanCut gated_scan_cut(int64_t B, int64_t T, int64_t C, bool backward) {
  constexpr int64_t unit = GS_W * GS_FWD_L;       // a segment is a multiple of it
  const int64_t blocks = B * ceil_div(C, (int64_t)64), sms = num_sms();
  int64_t segs = 1;
  if (blocks > 0 && blocks * (backward ? 2 : 3) < sms) segs = ceil_div(4 * sms, blocks);
  const int64_t most = T / (2 * unit);
  segs = segs < most ? segs : most;
  if (segs <= 1) return {1, ceil_div(T > 0 ? T : 1, unit) * unit};
  const int64_t len = ceil_div(ceil_div(T, segs), unit) * unit;
  return {(int)ceil_div(T, len), len};
}

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
