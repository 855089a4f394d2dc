// rowvec.cuh -- vectors of consecutive channels of a row, in fp32 or bf16
// storage, unpacked to fp32 registers: shared by the embedding and the
// residual-norm kernels (embedding.cu, residual_norm.cu).
#pragma once

#include "common.cuh"

namespace tp {

struct bf16_t {   // storage only
  uint16_t v;
};

__device__ __forceinline__ uint16_t f32_to_bf16_bits(float f) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(f));
}
// two rounded values in one word (first value in the low half); the cast of a
// pair is one instruction on sm_100a
__device__ __forceinline__ uint32_t f32x2_to_bf16x2_bits(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// VEC consecutive elements of type T as one load or store
template <typename T, int VEC>
struct RowVec;

template <>
struct RowVec<float, 4> {
  float4 r;
  __device__ __forceinline__ void zero() { r = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) {
    r = __ldg(reinterpret_cast<const float4*>(p));
  }
  __device__ __forceinline__ void load_stream(const float* p) {
    r = __ldcs(reinterpret_cast<const float4*>(p));
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w;
  }
  __device__ __forceinline__ void set(const float* f) { r = make_float4(f[0], f[1], f[2], f[3]); }
  __device__ __forceinline__ void pack(const float* e) { set(e); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<float4*>(p) = r; }
  __device__ __forceinline__ void store_stream(float* p) const {
    __stcs(reinterpret_cast<float4*>(p), r);
  }
};

template <>
struct RowVec<float, 2> {
  float2 r;
  __device__ __forceinline__ void zero() { r = make_float2(0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) {
    r = __ldg(reinterpret_cast<const float2*>(p));
  }
  __device__ __forceinline__ void load_stream(const float* p) {
    r = __ldcs(reinterpret_cast<const float2*>(p));
  }
  __device__ __forceinline__ void get(float* f) const { f[0] = r.x; f[1] = r.y; }
  __device__ __forceinline__ void set(const float* f) { r = make_float2(f[0], f[1]); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<float2*>(p) = r; }
  __device__ __forceinline__ void store_stream(float* p) const {
    __stcs(reinterpret_cast<float2*>(p), r);
  }
};

template <>
struct RowVec<float, 1> {
  float r;
  __device__ __forceinline__ void zero() { r = 0.f; }
  __device__ __forceinline__ void load(const float* p) { r = __ldg(p); }
  __device__ __forceinline__ void load_stream(const float* p) { r = __ldcs(p); }
  __device__ __forceinline__ void get(float* f) const { f[0] = r; }
  __device__ __forceinline__ void set(const float* f) { r = f[0]; }
  __device__ __forceinline__ void store(float* p) const { *p = r; }
  __device__ __forceinline__ void store_stream(float* p) const { __stcs(p, r); }
};

template <>
struct RowVec<bf16_t, 8> {
  uint4 r;
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const bf16_t* p) {
    r = __ldg(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void load_stream(const bf16_t* p) {
    r = __ldcs(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void get(float* f) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    r.x = f32x2_to_bf16x2_bits(f[0], f[1]);
    r.y = f32x2_to_bf16x2_bits(f[2], f[3]);
    r.z = f32x2_to_bf16x2_bits(f[4], f[5]);
    r.w = f32x2_to_bf16x2_bits(f[6], f[7]);
  }
  __device__ __forceinline__ void pack(const bf16_t* e) {
    r = make_uint4(e[0].v | (uint32_t)e[1].v << 16, e[2].v | (uint32_t)e[3].v << 16,
                   e[4].v | (uint32_t)e[5].v << 16, e[6].v | (uint32_t)e[7].v << 16);
  }
  __device__ __forceinline__ void store(bf16_t* p) const { *reinterpret_cast<uint4*>(p) = r; }
  __device__ __forceinline__ void store_stream(bf16_t* p) const {
    __stcs(reinterpret_cast<uint4*>(p), r);
  }
};

template <>
struct RowVec<bf16_t, 4> {
  uint2 r;
  __device__ __forceinline__ void zero() { r = make_uint2(0, 0); }
  __device__ __forceinline__ void load(const bf16_t* p) {
    r = __ldg(reinterpret_cast<const uint2*>(p));
  }
  __device__ __forceinline__ void load_stream(const bf16_t* p) {
    r = __ldcs(reinterpret_cast<const uint2*>(p));
  }
  __device__ __forceinline__ void get(float* f) const {
    const uint32_t w[2] = {r.x, r.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    r.x = f32x2_to_bf16x2_bits(f[0], f[1]);
    r.y = f32x2_to_bf16x2_bits(f[2], f[3]);
  }
  __device__ __forceinline__ void store(bf16_t* p) const { *reinterpret_cast<uint2*>(p) = r; }
  __device__ __forceinline__ void store_stream(bf16_t* p) const {
    __stcs(reinterpret_cast<uint2*>(p), r);
  }
};

template <>
struct RowVec<bf16_t, 2> {
  uint32_t r;
  __device__ __forceinline__ void zero() { r = 0; }
  __device__ __forceinline__ void load(const bf16_t* p) {
    r = __ldg(reinterpret_cast<const unsigned int*>(p));
  }
  __device__ __forceinline__ void load_stream(const bf16_t* p) {
    r = __ldcs(reinterpret_cast<const unsigned int*>(p));
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = __uint_as_float(r << 16);
    f[1] = __uint_as_float(r & 0xffff0000u);
  }
  __device__ __forceinline__ void set(const float* f) { r = f32x2_to_bf16x2_bits(f[0], f[1]); }
  __device__ __forceinline__ void store(bf16_t* p) const { *reinterpret_cast<uint32_t*>(p) = r; }
  __device__ __forceinline__ void store_stream(bf16_t* p) const {
    __stcs(reinterpret_cast<unsigned int*>(p), r);
  }
};

template <>
struct RowVec<bf16_t, 1> {
  uint16_t r;
  __device__ __forceinline__ void zero() { r = 0; }
  __device__ __forceinline__ void load(const bf16_t* p) {
    r = __ldg(reinterpret_cast<const unsigned short*>(p));
  }
  __device__ __forceinline__ void load_stream(const bf16_t* p) {
    r = __ldcs(reinterpret_cast<const unsigned short*>(p));
  }
  __device__ __forceinline__ void get(float* f) const { f[0] = tp_bf16_to_f32(r); }
  __device__ __forceinline__ void set(const float* f) { r = f32_to_bf16_bits(f[0]); }
  __device__ __forceinline__ void store(bf16_t* p) const {
    *reinterpret_cast<uint16_t*>(p) = r;
  }
  __device__ __forceinline__ void store_stream(bf16_t* p) const {
    __stcs(reinterpret_cast<unsigned short*>(p), r);
  }
};

__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// sigmoid(v) and 1 - sigmoid(v), both to fp32 accuracy: with e = exp(-|v|) the
// smaller one is e / (1 + e), with no cancellation and no overflow (NaN stays NaN),
// and the larger one is 1 less that.  The quotient 1 / (1 + e) instead is off by up to
// an ulp, always to the same side for like arguments: a gate of a long memory applies
// that error once a step (h_last of 1536 steps at gates around sigmoid(6): root mean
// square error 2.8 times that of correctly rounded gates).
__device__ __forceinline__ void sigmoid_pair(float v, float& s, float& rest) {
  const float e = expf(-fabsf(v));
  const float small = e * rcp_approx(1.0f + e);
  const float big = 1.0f - small;
  s = v >= 0.0f ? big : small;
  rest = v >= 0.0f ? small : big;
}

// The same for bf16 storage: e = exp(-v) as one power of two.  Relative error of
// what comes from it about (8 + 1.5 |v|) 2^-24 (argument rounded once, 2^x to
// 2^-22, 1 + e, reciprocal and product); a gate above 1/2 is 1 less its complement,
// off by that of the complement and a rounding.  The exponent is held at 126, so that
// sigmoid(-inf) is 2^-126 and its complement exactly 1.
__device__ __forceinline__ float ex2_of_capped(float t) {
  asm("min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(t));   // 126
  return tp_ex2(t);
}
__device__ __forceinline__ void fast_sigmoid_pair(float v, float& s, float& rest) {
  const float e = ex2_of_capped(__fmul_rn(v, -1.442695041f));
  const float r = rcp_approx(__fadd_rn(1.0f, e));
  rest = __fmul_rn(e, r);
  const float big = __fsub_rn(1.0f, rest);
  s = v > 0.0f ? big : r;
}
// two at once, the same bits
__device__ __forceinline__ void fast_sigmoid_pair2(float2 v, float2& s, float2& rest) {
  const float2 one = make_float2(1.0f, 1.0f);
  const float2 t = tp_mul2(v, make_float2(-1.442695041f, -1.442695041f));
  const float2 e = make_float2(ex2_of_capped(t.x), ex2_of_capped(t.y));
  const float2 d = tp_add2(one, e);
  const float2 r = make_float2(rcp_approx(d.x), rcp_approx(d.y));
  rest = tp_mul2(e, r);
  const float2 big = tp_fma2(rest, make_float2(-1.0f, -1.0f), one);
  s = make_float2(v.x > 0.0f ? big.x : r.x, v.y > 0.0f ? big.y : r.y);
}

}  // namespace tp
