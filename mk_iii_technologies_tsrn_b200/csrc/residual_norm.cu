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
// writes dx, dbranch, dgate.  A team of G threads (a warp, or a block of up to
// 16 warps for long rows) holds a whole row in registers, so the statistics cost
// no second read; all loads of a row are issued before the first use, and the
// team's next row is asked into L2 meanwhile.  The backward recomputes y from x
// (the same bytes as reading y, and exact where the stored y is rounded to bf16)
// and takes the row statistics (mean and 1 / deviation of y and branch) from the
// forward.
//
// Rows of an odd length begin inside 16 bytes, each at another element; rows
// eight apart begin at the same one.  So a block takes rows that are alike modulo
// eight, and its vectors lie on 16 bytes in all of them, each with channels of its
// own for good (the column sums need that): only the first and the last vector of
// a row are cut.  42919 x 1031 bf16: 168 and 372 us against 594 and 1199 us with
// single channels.
//
// Parameter gradients are column sums.  Up to five of them run at once (w, b,
// channel scale, bw, bb), too many to stay in registers beside the row, so
// each thread keeps those of its own columns in shared memory (16-byte
// read-add-writes without conflicts, no synchronisation); a block adds its
// teams in order and a second kernel adds the blocks in order, so the same
// inputs give the same bits.  A single scale's gradient is one sum over all
// elements, whose terms may cancel: a row of it is added in fp32, the rows in
// 64 bits.
//
// Measured (forward, backward), in the bytes above: 65536 x 640 fp32 with gate and
// LayerNorm 139 us (6.0 TB/s) and 241 us (5.6); 16384 x 2048 fp32 with a branch
// norm and a channel scale 94 (5.7) and 200 us (4.0), bf16 59 (4.5) and 159 us
// (2.5): bf16 rows have the same arithmetic for half the bytes, and the backward's
// 128 registers a thread leave 16 warps on an SM to hide it.
#include <initializer_list>

#include "residual_norm.cuh"

namespace tp {

namespace {

// Column sums over the blocks' partials, in block order: 32 columns per block,
// 8 warps each take a contiguous range of the partials.  The last block adds the
// single scale's, in 64 bits.
__global__ void __launch_bounds__(256) residual_norm_sum_kernel(const ResNormBwdArgs g,
                                                                int blocks) {
  __shared__ float s[8][32];
  const int64_t columns = (int64_t)g.sums * g.f.D, width = columns + 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x == gridDim.x - 1) {
    if (g.f.scale_mode != 1 || g.dscale == nullptr || warp != 0) return;
    double t = 0.0;
    for (int i = lane; i < blocks; i += 32)
      t += (double)g.part[(int64_t)i * width + columns] +
           (double)g.part[(int64_t)i * width + columns + 1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) *g.dscale = (float)t;
    return;
  }
  const int64_t col = (int64_t)blockIdx.x * 32 + lane;
  const int per = (blocks + 7) / 8;
  const int lo = warp * per, hi = min(blocks, lo + per);
  float acc = 0.f;
  if (col < columns) {
#pragma unroll 8
    for (int i = lo; i < hi; ++i) acc += g.part[(int64_t)i * width + col];
  }
  s[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || col >= columns) return;
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += s[w][lane];
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
  bool known;       // gate, branch norm and parameters known at compile time
  bool warp;        // a team is a warp, else a block
  bool shift;       // rows begin inside 16 bytes
  bool staged;      // parameters in shared memory
};

// Vectors per thread and threads per row.  A warp as long as its registers hold
// the row (20 fp32 or 24 bf16 elements per thread), else a block of whole warps
// around it (16 elements per thread, 8 of fp32 rows that begin inside 16 bytes).
Plan plan_row(bool bf16, bool shift, int vec, int64_t D, bool params_f32) {
  Plan p;
  p.vec = vec;
  p.shift = shift;
  const int64_t n = shift ? shifted_vectors((int)D, vec) : ceil_div(D, (int64_t)vec);
  p.warp = vec == (bf16 ? 8 : 4) && n <= 32 * (bf16 ? 3 : 5);
  p.staged = p.warp || shift;
  if (p.warp) {
    p.known = true;
    p.group = 32;
    p.nv = (int)ceil_div(n, (int64_t)32);
    if (shift && p.nv % 2 == 0) ++p.nv;      // 1, 3 or 5
    return p;
  }
  p.known = shift || (params_f32 && vec > 1);
  p.nv = shift && !bf16 ? 2 : 16 / vec;
  p.group = (int)ceil_div(ceil_div(n, (int64_t)p.nv), (int64_t)32) * 32;
  // (the dispatch tells warps by a group of 32: a block of one warp takes two)
  if (p.known && p.group == 32) p.group = 64;
  return p;
}

// vectors of rows that begin on a vector's bytes
bool vec_ok(const ResNormArgs& a, int vec, int esize) {
  const int64_t m = (int64_t)vec * esize - 1;   // 8- or 16-byte vectors
  auto al = [&](const void* q) { return q == nullptr || (((uintptr_t)q) & m) == 0; };
  auto al16 = [](const void* q) { return q == nullptr || aligned16(q); };
  return a.D % vec == 0 && al(a.x) && al(a.branch) && al(a.gate) && al(a.y) && al(a.n) &&
         a.ldx % vec == 0 && a.ldb % vec == 0 && (a.gate == nullptr || a.ldg % vec == 0) &&
         al16(a.w) && al16(a.b) && al16(a.bw) && al16(a.bb) &&
         (a.scale_mode != 2 || al16(a.scale));
}
// and of rows whose first channels lie at the same element of 16 bytes in all tensors.
// (The 512 threads of two fp32 vectors reach over 4093 channels at any shift.)
bool shift_ok(const ResNormArgs& a, int vec) {
  auto al = [](const void* q) { return q == nullptr || aligned16(q); };
  auto ld = [&](int64_t l) { return l >= a.D && l % vec == a.D % vec; };
  return a.D <= 4080 && a.D % RN_RESIDUES != 0 && al(a.x) && al(a.branch) && al(a.gate) && al(a.y) && al(a.n) &&
         ld(a.ldx) && ld(a.ldb) && (a.gate == nullptr || ld(a.ldg));
}

int common_align(std::initializer_list<const void*> ps) {
  uintptr_t m = 16;
  for (const void* q : ps) m |= (uintptr_t)q;
  return (int)(m & (~m + 1));
}

Plan plan(const ResNormArgs& a, int align_of_grads) {
  const bool bf16 = a.dtype == TP_DTYPE_BF16;
  const int esize = bf16 ? 2 : 4;
  for (int vec : {bf16 ? 8 : 4, 4})
    if (align_of_grads % (vec * esize) == 0 && vec_ok(a, vec, esize))
      return plan_row(bf16, false, vec, a.D, !a.params_bf16);
  if (align_of_grads == 16 && shift_ok(a, 16 / esize))
    return plan_row(bf16, true, 16 / esize, a.D, !a.params_bf16);
  return plan_row(bf16, false, 1, a.D, !a.params_bf16);
}

size_t staged_bytes(const ResNormArgs& a, const Plan& p, bool backward) {
  if (!p.staged) return 0;
  const int n = (a.w != nullptr) + (!backward && a.b != nullptr) + (a.scale_mode == 2) +
                (a.bw != nullptr) + (a.bb != nullptr);
  return sizeof(float) * (size_t)n * (p.shift ? staged_size((int)a.D, p.vec) : (int)a.D);
}

// the kernels that look everything up: other alignments, bf16 parameters of long rows
template <typename T, int VEC>
int fwd_any(const ResNormArgs& a, cudaStream_t s) {
  return launch_fwd_kernel<T, VEC, 16 / VEC, 0, RN_ANY, 2, 2, false>(a, 0, s);
}
template <typename T, int VEC>
int bwd_any(const ResNormBwdArgs& g, size_t smem, int blocks, cudaStream_t s) {
  return launch_bwd_kernel<T, VEC, 16 / VEC, 0, RN_ANY, 2, 2, false>(g, smem, blocks, s);
}

}  // namespace

bool residual_norm_supported(int64_t D) { return D >= 1 && D <= 8192; }

int residual_norm_bwd_blocks(int64_t rows, int64_t D) {
  // what an SM holds at once: three blocks of four rows, or rows in 512 threads of
  // 128 registers.  Each block keeps a set of column sums, so more than four only where
  // each then still has 16 rows.  Rows that may begin inside 16 bytes want a multiple of
  // the residues.
  const int64_t threads = ceil_div(D, (int64_t)512) * 32;
  int64_t per_sm = D <= 640 ? 3 : (threads <= 256 ? 512 / threads : 1);
  if (per_sm > 4 && rows < 16 * per_sm * num_sms()) per_sm = 4;
  const int64_t r = D % RN_RESIDUES ? RN_RESIDUES : 1;
  const int64_t cap = (int64_t)num_sms() * per_sm / r * r;
  const int64_t want = ceil_div(rows > 0 ? rows : 1, r) * r;
  return (int)(want < cap ? want : cap);
}

int launch_residual_norm_fwd(const ResNormArgs& args, cudaStream_t stream) {
  ResNormArgs a = args;
  const bool bf16 = a.dtype == TP_DTYPE_BF16;
  const Plan p = plan(a, 16);
  a.group = p.group;
  const size_t smem = staged_bytes(a, p, false);
  if (p.shift) return launch_residual_norm_fwd_shift(p.nv, a, smem, stream);
  if (p.known)
    return bf16 ? launch_residual_norm_fwd_bf16(p.vec, p.nv, a, smem, stream)
                : launch_residual_norm_fwd_f32(p.vec, p.nv, a, smem, stream);
  if (!bf16) return p.vec == 4 ? fwd_any<float, 4>(a, stream) : fwd_any<float, 1>(a, stream);
  if (p.vec == 8) return fwd_any<bf16_t, 8>(a, stream);
  return p.vec == 4 ? fwd_any<bf16_t, 4>(a, stream) : fwd_any<bf16_t, 1>(a, stream);
}

int launch_residual_norm_bwd(const ResNormBwdArgs& args, cudaStream_t stream) {
  ResNormBwdArgs g = args;
  const bool bf16 = g.f.dtype == TP_DTYPE_BF16;
  int k = 0;
  g.slot_w = g.dw ? k++ : -1;
  g.slot_b = g.db ? k++ : -1;
  g.slot_s = (g.f.scale_mode == 2 && g.dscale) ? k++ : -1;
  g.slot_bw = g.dbw ? k++ : -1;
  g.slot_bb = g.dbb ? k++ : -1;
  g.sums = k;
  int blocks = residual_norm_bwd_blocks(g.f.rows, g.f.D);
  const Plan p = plan(g.f, common_align({g.dy, g.dn, g.dx, g.dbranch, g.dgate}));
  g.f.group = p.group;
  const size_t smem = sizeof(float) * (size_t)k * p.vec * p.nv * (p.warp ? 128 : p.group) +
                      staged_bytes(g.f, p, true);
  int st;
  // one wave, where rows take more threads than that count supposes
  const int r = p.shift ? RN_RESIDUES : 1;
  const int fit = num_sms() * (p.warp ? 3 : max(512 / p.group, 1)) / r * r;
  blocks = min(blocks, fit);
  if (p.shift) {
    st = bf16 ? launch_residual_norm_bwd_shift_bf16(p.nv, g, smem, blocks, stream)
              : launch_residual_norm_bwd_shift_f32(p.nv, g, smem, blocks, stream);
  } else if (p.known) {
    st = bf16 ? launch_residual_norm_bwd_bf16(p.vec, p.nv, g, smem, blocks, stream)
              : launch_residual_norm_bwd_f32(p.vec, p.nv, g, smem, blocks, stream);
  } else if (!bf16) {
    st = p.vec == 4 ? bwd_any<float, 4>(g, smem, blocks, stream)
                    : bwd_any<float, 1>(g, smem, blocks, stream);
  } else if (p.vec == 8) {
    st = bwd_any<bf16_t, 8>(g, smem, blocks, stream);
  } else {
    st = p.vec == 4 ? bwd_any<bf16_t, 4>(g, smem, blocks, stream)
                    : bwd_any<bf16_t, 1>(g, smem, blocks, stream);
  }
  if (st != TP_OK) return st;
  const unsigned sum_blocks = (unsigned)ceil_div((int64_t)k * g.f.D, (int64_t)32) + 1;
  residual_norm_sum_kernel<<<sum_blocks, 256, 0, stream>>>(g, blocks);
  return launch_status();
}

}  // namespace tp
