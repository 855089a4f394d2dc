// paged_attention_bf16.cu -- paged attention over bf16 caches: on the tensor cores where rows
// begin and end on 16 bytes, but for blended scores (paged_attention.cuh).
//
// The products are 8 query heads by the slots, so m16n8k16 instructions of one warp: eight of
// their sixteen rows are heads, and there is nothing to gain from tcgen05's 128 rows -- the
// kernel waits for DRAM.  Rows of K and V are copied whole and in their order, and read from
// shared memory as the instructions' operands lie in the lanes (every lane copying what its own
// operands need instead asks for 32 bytes of a line at a time):
//   S = Q K^T: the contraction runs over the channels in any order that Q and K share, so lane
//     (g, t) takes channels 8t .. 8t + 7 of each 32 of a slot (and of head g of Q).
//   O = P V: P is where S was left.  Lane (g, t) takes channels 8g .. 8g + 7 of each 64 of the
//     four slots whose weights it holds; pairs of slots are interleaved in registers.
// Every second row is moved on by 32 bytes, and column g of the eight slots of an instruction is
// slot `slot_of(g)`, so that neither read meets a bank twice.
// A weight is a sum of bf16 parts (products of two bf16 numbers are exact in fp32).  Blocks of up to
// four query heads have each head in rows g and g + 4 of S, so that P's rows g, g + 8 and g + 4 take
// its three parts: all 24 bits (48 x 8192 of 4 query heads each 198.7 us for 197.7 with two parts, of one
// head of 64 channels 106 for 107.5).  Blocks of five to eight have rows g and g + 8 alone: two parts,
// which lose at most 2^-16 of a weight, where the output is rounded by 2^-8 (a second product for the
// other bits: 24 x 8192 of 16 query heads each 95 -> 105 us, 48 x 8192 of 8 heads of 64 115 -> 122).
// So do all above 192 channels, whose registers are full (48 x 4096 of 4 heads of 256 channels 249 us,
// 286 with three parts).  Everything else is fp32.
#include "paged_attention.cuh"

namespace tp {

namespace {

// D += A B, A 16 x 16 and B 16 x 8 of bf16
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *(const uint32_t*)&p;
}

// KB blocks of 32 channels
template <int KB>
struct MmaTile {
  static constexpr int VB = (KB + 1) / 2;                    // blocks of 64 channels
  static constexpr int PIECES = KB <= 2 ? 8 : KB <= 4 ? 16 : 32;      // of 16 bytes, of a row
  static constexpr int GROUPS = KB <= 2 ? 2 : 1;             // of 16 slots
  static constexpr int TK = 16 * GROUPS;
  static constexpr int ROWS = 32 / PIECES, STEPS = TK / ROWS;         // of a copy; copies of K
  static constexpr int HALF = TK * PIECES + TK;              // 16-byte pieces of K, and of V
  static constexpr int STAGE = 2 * HALF;                     // of a warp's stage
};
// where a slot's row begins, in pieces of 16 bytes
template <int PIECES>
__device__ __forceinline__ constexpr int row_at(int slot) {
  return slot * PIECES + slot / 2 * 2;
}
// 0 4 2 6 5 1 7 3: of an even column and the next one, 64 bytes apart modulo 128; the even columns,
// and the odd ones, 32 apart
__device__ __forceinline__ int slot_of(int column) {
  const int t = column >> 1, even = 2 * t + (t >> 1);
  return column & 1 ? even ^ 4 : even;
}

// The copies of a tile: step S has slots S * ROWS + (the lane's).
template <typename P, int S = 0>
__device__ __forceinline__ void copy_rows(uint32_t to, const char* const (&kfrom)[P::STEPS],
                                          const char* const (&vfrom)[P::STEPS]) {
  // (one row a copy: rows 2i + 1 lie PIECES behind rows 2i)
  constexpr int AT = 16 * row_at<P::PIECES>(S * P::ROWS);
  copy16<AT, 0>(to, kfrom[S]);
  copy16<P::HALF * 16 + AT, 0>(to, vfrom[S]);
  if constexpr (S + 1 < P::STEPS) copy_rows<P, S + 1>(to, kfrom, vfrom);
}

// FEW: blocks of up to four query heads
template <int KB, int STAGES, bool FEW>
__global__ void __launch_bounds__(ATT_WARPS * 32) paged_attend_mma_kernel(const PagedAttentionArgs a) {
  using P = MmaTile<KB>;
  constexpr int HEADS = FEW ? 4 : 8;
  constexpr int VB = P::VB, GROUPS = P::GROUPS, TK = P::TK;
  extern __shared__ __align__(128) char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int D = a.c.channels, subs = a.c.heads * a.head_blocks;
  const int64_t mine = (int64_t)blockIdx.x * ATT_WARPS + warp;
  const int run = (int)(mine / subs), hsub = (int)(mine - (int64_t)run * subs);
  const int kvh = hsub / a.head_blocks, hblk = hsub - kvh * a.head_blocks;
  int count;
  Place at = place_of_run<TK>(a, run, count);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (count == 0) return;

  uint4* const ring = (uint4*)smem + (size_t)warp * STAGES * P::STAGE;
  const int pieces = D / 8, row = lane / P::PIECES, piece = lane % P::PIECES;
  const bool copies = piece < pieces;
  const int mine_at = 16 * (row_at<P::PIECES>(row) + piece);      // of this lane's pieces
  if (pieces < P::PIECES)                  // channels that are not there: zeros, never copied to
    for (int i = lane; i < STAGES * P::STAGE; i += 32) ring[i] = make_uint4(0, 0, 0, 0);
  __syncwarp();

  Place ahead = at;
  TileRows<uint16_t, TK> rows(a, kvh);
  rows.ask(ahead);
  // (this lane's piece of its first row in page 0, and from one of its rows to the next)
  const int64_t k_step = P::ROWS * a.c.k_slot, v_step = P::ROWS * a.c.v_slot;
  const char* const kmine = a.c.k + (int64_t)kvh * a.c.k_head + row * a.c.k_slot + piece * 16;
  const char* const vmine = a.c.v + (int64_t)kvh * a.c.v_head + row * a.c.v_slot + piece * 16;
  auto issue = [&](int i) {
    if (i < count) {
      const uint32_t to = tp_smem_addr(ring + (size_t)(i % STAGES) * P::STAGE) + mine_at;
      const char *kp, *vp, *kfrom[P::STEPS], *vfrom[P::STEPS];
      if (rows.in_halves(ahead)) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          int64_t k_at, v_at;
          rows.half_at(ahead, half, k_at, v_at);
          kp = kmine + k_at;
          vp = vmine + v_at;
#pragma unroll
          for (int s = half * P::STEPS / 2; s < (half + 1) * P::STEPS / 2; ++s, kp += k_step, vp += v_step) {
            kfrom[s] = kp;
            vfrom[s] = vp;
          }
        }
      } else {
        rows.get(ahead, kp, vp);
#pragma unroll
        for (int s = 0; s < P::STEPS; ++s) {
          kfrom[s] = shfl_ptr(kp, s * P::ROWS + row) + piece * 16;
          vfrom[s] = shfl_ptr(vp, s * P::ROWS + row) + piece * 16;
        }
      }
      if (copies) copy_rows<P>(to, kfrom, vfrom);
      if (i + 1 < count) {
        forward<TK>(a, ahead);
        rows.ask(ahead);
      }
    }
    tp_cp_async_commit();
  };

  const int kslot = slot_of(g), slot0 = slot_of(2 * t);      // of each eight; slot0 ^ 4: column 2t + 1
  uint4 q[KB];
  const int head = FEW ? g & 3 : g;        // of the block: this lane's
  float factor = 0.0f, m = neg_inf(), l = 0.0f;      // of that head; l: the sum of this lane's slots
  int h = 0;
  bool head_there = false, writes = false;
  float acc[VB][8][4];
  auto begin_row = [&]() {
    const int in_group = hblk * HEADS + head;
    head_there = in_group < a.group;
    writes = head_there && head == g;
    h = kvh * a.group + (head_there ? in_group : 0);
    const uint16_t* src = (const uint16_t*)a.q + (int64_t)at.b * a.q_sb + (int64_t)h * a.q_sh;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      alignas(16) uint16_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = head_there && kb * 32 + t * 8 < D ? __ldg(src + kb * 32 + t * 8 + i) : (uint16_t)0;
      q[kb] = *(const uint4*)e;
    }
    factor = (a.tau ? a.scale / __ldg(a.tau + h) : a.scale) * 1.4426950408889634f;
    m = neg_inf();
    l = 0.0f;
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[vb][j][i] = 0.0f;
  };
  auto end_row = [&]() {               // the segment
    const int64_t seg = segment(a, at.b, run, hsub);
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* const to = a.part + (seg * HEADS + head) * D + 16 * t;
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float most = acc[vb][j][e];
          float rest = acc[vb][j][2 + e];
          if constexpr (FEW) rest += __shfl_xor_sync(0xffffffffu, most, 16);      // (of row g + 4)
          // (an infinite value makes NaN of the lesser parts, which may be 0 or of the other sign)
          x[j] = fabsf(most) < -neg_inf() ? most + rest : most;
        }
        if (writes && vb * 64 + 16 * t + 8 * e < D) {
          float4* const at4 = (float4*)(to + vb * 64 + 8 * e);
          at4[0] = make_float4(x[0], x[1], x[2], x[3]);
          at4[1] = make_float4(x[4], x[5], x[6], x[7]);
        }
      }
    if (writes && t == 0) a.ml[seg * HEADS + head] = make_float2(m, l);
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i);
  bool fresh = true;
  for (int i = 0; i < count; ++i) {
    __syncwarp();                          // the tile before has been read by all lanes
    issue(i + STAGES - 1);
    if (fresh) begin_row();
    tp_cp_async_wait<STAGES - 1>();
    __syncwarp();                          // the tile is there, all lanes' pieces
    const uint4* kst = ring + (size_t)(i % STAGES) * P::STAGE;
    const uint4* vst = kst + P::HALF;
    const uint4* const kmid = kst + row_at<P::PIECES>(kslot) + t;
    const uint4* const v0mid = vst + row_at<P::PIECES>(slot0) + g;
    const uint4* const v1mid = vst + row_at<P::PIECES>(slot0 ^ 4) + g;
    const int base = at.tile * TK, n = at.n;

    float s[2 * GROUPS][2];                 // head g, columns 2t and 2t + 1 of eight slots
    float top = neg_inf();
#pragma unroll
    for (int j = 0; j < 2 * GROUPS; ++j) {
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint4 k = kmid[row_at<P::PIECES>(8 * j) + kb * 4];
        mma16816(c, q[kb].x, 0u, q[kb].y, 0u, k.x, k.y);
        mma16816(c, q[kb].z, 0u, q[kb].w, 0u, k.z, k.w);
      }
      const int at0 = base + 8 * j + slot0, at1 = base + 8 * j + (slot0 ^ 4);
      s[j][0] = at0 < n ? c[0] * factor : neg_inf();
      s[j][1] = at1 < n ? c[1] * factor : neg_inf();
      top = fmaxf(top, fmaxf(s[j][0], s[j][1]));
      if (a.scores != nullptr && writes) {
        float* sc = a.scores + ((int64_t)at.b * a.H + h) * a.score_row;
        if (at0 < n) sc[at0] = s[j][0];
        if (at1 < n) sc[at1] = s[j][1];
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float to = fmaxf(m, top), from = to == neg_inf() ? 0.0f : to;
    if (__any_sync(0xffffffffu, to != m)) {
      const float less = to == m ? 1.0f : tp_ex2(m - from);
      l *= less;
#pragma unroll
      for (int vb = 0; vb < VB; ++vb)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[vb][j][x] *= less;
      m = to;
    }
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) {
      uint32_t p[4];                       // parts of slots 2t, 2t + 1 of two eights, rows g and g + 8
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float p0 = tp_ex2(s[2 * u + e][0] - from), p1 = tp_ex2(s[2 * u + e][1] - from);
        l += p0 + p1;
        if constexpr (FEW) {
          auto part = [&]() {              // the first 8 bits, cut off; what is left is exact
            const uint32_t x0 = __float_as_uint(p0), x1 = __float_as_uint(p1);
            p0 -= __uint_as_float(x0 & 0xffff0000u);
            p1 -= __uint_as_float(x1 & 0xffff0000u);
            return __byte_perm(x0, x1, 0x7632);
          };
          const uint32_t first = part(), second = part(), third = part();
          p[2 * e] = head == g ? first : third;
          p[2 * e + 1] = head == g ? second : 0u;
        } else {
          const uint32_t hi = pack_bf16(p0, p1);
          p[2 * e] = hi;
          p[2 * e + 1] = pack_bf16(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u));
        }
      }
#pragma unroll
      for (int vb = 0; vb < VB; ++vb) {
        constexpr int EIGHT = row_at<P::PIECES>(8);
        const uint4 v0 = v0mid[2 * u * EIGHT + vb * 8], v1 = v1mid[2 * u * EIGHT + vb * 8],
                    v2 = v0mid[(2 * u + 1) * EIGHT + vb * 8], v3 = v1mid[(2 * u + 1) * EIGHT + vb * 8];
        const uint32_t x0[4] = {v0.x, v0.y, v0.z, v0.w}, x1[4] = {v1.x, v1.y, v1.z, v1.w},
                       x2[4] = {v2.x, v2.y, v2.z, v2.w}, x3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t pick = j & 1 ? 0x7632 : 0x5410;
          mma16816(acc[vb][j], p[0], p[1], p[2], p[3], __byte_perm(x0[j / 2], x1[j / 2], pick),
                   __byte_perm(x2[j / 2], x3[j / 2], pick));
        }
      }
    }
    fresh = at.tile + 1 == at.tiles || i + 1 == count;
    if (fresh) end_row();
    if (i + 1 < count) forward<TK>(a, at);
  }
  tp_cp_async_wait<0>();
}

template <int KB>
int attend_mma(PagedAttentionArgs& a, cudaStream_t stream) {
  constexpr int STAGES = KB > 4 ? 2 : 3;
  using P = MmaTile<KB>;
  const size_t smem = (size_t)ATT_WARPS * STAGES * P::STAGE * 16;
  if constexpr (KB <= 6)
    if (a.group <= 4)
      return attend_and_join<uint16_t>(a, paged_attend_mma_kernel<KB, STAGES, true>, smem, P::TK, 4, stream);
  return attend_and_join<uint16_t>(a, paged_attend_mma_kernel<KB, STAGES, false>, smem, P::TK, 8, stream);
}

int on_tensor_cores(PagedAttentionArgs& a, cudaStream_t stream) {
  const int D = a.c.channels;
  return D <= 32    ? attend_mma<1>(a, stream)
         : D <= 64  ? attend_mma<2>(a, stream)
         : D <= 96  ? attend_mma<3>(a, stream)
         : D <= 128 ? attend_mma<4>(a, stream)
         : D <= 192 ? attend_mma<6>(a, stream)
                    : attend_mma<8>(a, stream);
}

template <int LPK>
int on_cores(PagedAttentionArgs& a, bool vec, cudaStream_t stream) {
  if (!vec)
    return a.gate ? attend<uint16_t, LPK, 1, 1, true, false>(a, stream)
                  : attend<uint16_t, LPK, 1, 1, false, false>(a, stream);
  return a.group == 1   ? attend<uint16_t, LPK, 1, 1, true, true>(a, stream)
         : a.group == 2 ? attend<uint16_t, LPK, 1, 2, true, true>(a, stream)
                        : attend<uint16_t, LPK, 1, 4, true, true>(a, stream);
}

}  // namespace

int launch_paged_attention_bf16(PagedAttentionArgs a, bool vec, cudaStream_t stream) {
  const int D = a.c.channels;
  return vec && a.gate == nullptr ? on_tensor_cores(a, stream)
         : D <= 64                ? on_cores<8>(a, vec, stream)
         : D <= 128               ? on_cores<16>(a, vec, stream)
                                  : on_cores<32>(a, vec, stream);
}

}  // namespace tp
