// The 8-bit format shared by the quantising operators and their readers.
//
// A group of values v (a whole row, or 128 columns of a checkpoint) is held as
// int8 codes and one fp32 scale:
//
//   a = max(max|v|, 2^-110),  q = rint(v * (127 / a)),  scale = a / 127,  v ~ q * scale
//
// with IEEE fp32 divisions and product, so the codes of a group do not depend
// on how the group is split over threads.  |q| <= 127: 127 / a and the product
// are each at most (1 + 2^-24) too large, and 127 (1 + 2^-24)^2 rounds to 127.
// The floor 2^-110 keeps 127 / a and a / 127 normal numbers; smaller groups
// read back as multiples of 2^-110 / 127.  A group that holds an infinity or a
// NaN has scale NaN and codes 0: everything read back from it is NaN.
#pragma once

#include "hlm_common.cuh"

namespace hlm {

constexpr float kQuantFloor = 7.7037197775489434e-34f;  // 2^-110
constexpr uint32_t kInfBits = 0x7f800000u;
constexpr int kCkptGroup = 128;  // columns of one checkpoint group

// Magnitude of v as bits: ordered like the magnitudes, with infinities above
// every finite value and NaNs above infinity, so an integer maximum keeps both.
HLM_DEVICE uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct QuantStep {
  float inv;    // 127 / a, or 0 for a group that is not finite
  float scale;  // a / 127, or NaN
};
HLM_DEVICE QuantStep quant_step(uint32_t max_bits) {
  QuantStep s;
  if (max_bits >= kInfBits) {
    s.inv = 0.0f;
    s.scale = __uint_as_float(0x7fc00000u);
  } else {
    const float a = fmaxf(__uint_as_float(max_bits), kQuantFloor);
    s.inv = __fdiv_rn(127.0f, a);
    s.scale = __fdiv_rn(a, 127.0f);
  }
  return s;
}

// One of the two quotients of quant_step, for threads that share their maximum: each
// divides once, for the scale or for the inverse, and they pass the values on by shuffle.
HLM_DEVICE float quant_quotient(uint32_t max_bits, bool is_inv) {
  const float a = fmaxf(__uint_as_float(max_bits), kQuantFloor);
  const float d = __fdiv_rn(is_inv ? 127.0f : a, is_inv ? a : 127.0f);
  if (max_bits >= kInfBits) return is_inv ? 0.0f : __uint_as_float(0x7fc00000u);
  return d;
}

// Code of v.  rint through the fp32 magic number 1.5 * 2^23: for |v * inv| <= 127.0001
// the sum's low mantissa bits are the rounded (half to even) integer in two's
// complement, so the low byte of the sum is the code.  The product is rounded
// to fp32 first (no fused multiply-add), as the format defines it.  With inv = 0,
// an infinity or NaN in v gives NaN bits whose low byte is replaced by 0.
HLM_DEVICE uint32_t quant_bits(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f));
}
HLM_DEVICE int8_t quant_code(float v, const QuantStep& s) {
  return s.inv == 0.0f ? static_cast<int8_t>(0) : static_cast<int8_t>(quant_bits(v, s.inv) & 0xffu);
}
// Two floats rounded to a packed pair of 16-bit values, low half first.
template <typename T>
HLM_DEVICE uint32_t pack2(float a, float b);
template <>
HLM_DEVICE uint32_t pack2<__nv_bfloat16>(float a, float b) {
  return pack_bf16x2(a, b);
}
template <>
HLM_DEVICE uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Pairs of fp32 values in one register pair: sm_100 computes both with one instruction,
// each rounded as the single operation.  (A packed product that feeds a packed sum
// is contracted to a fused multiply-add, so products that have to be rounded first
// are summed one by one.)
struct F2 {
  uint64_t v;
};
HLM_DEVICE F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
HLM_DEVICE F2 f2(float x) { return f2(x, x); }
HLM_DEVICE void f2_split(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
HLM_DEVICE F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
HLM_DEVICE F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
HLM_DEVICE F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// 1 / (1 + 2^(-x log2 e)) of both values: the bits of sigmoid_fast, whose divide of 1 by a
// number not below 1 is the approximate reciprocal.  The argument is a rounded product with a
// rounded constant, so a value for negative x is off by up to 2 |x| 2^-24 of itself and a few
// units: below the rounding of 16-bit results, not of fp32 ones.  The forward uses it for fp32 too,
// since its output has the bits of the SwiGLU kernel, which does.
HLM_DEVICE F2 f2_sigmoid(F2 x) {
  float a, b;
  f2_split(x * f2(-1.4426950408889634f), a, b);
  f2_split(f2(ex2_ftz(a), ex2_ftz(b)) + f2(1.0f), a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return f2(a, b);
}

// For fp32 gradients: sigmoid(x) and 1 - sigmoid(x), each to some 2^-21 of itself whatever x.
// The complement is made from the exponential where the difference would cancel.
HLM_DEVICE void sigmoid_exact(float x, float& s, float& rest) {
  const float e = expf(-x);
  s = __fdividef(1.0f, 1.0f + e);
  rest = x < 0.0f ? 1.0f - s : e * s;
}

// Two packed 16-bit values, or two fp32 ones, as a pair (exact).
template <typename T>
HLM_DEVICE F2 f2_unpack(uint32_t w);
template <>
HLM_DEVICE F2 f2_unpack<__nv_bfloat16>(uint32_t w) {
  return f2(bf16_lo(w), bf16_hi(w));
}
template <>
HLM_DEVICE F2 f2_unpack<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f2(f.x, f.y);
}
// The pairs of a 16-byte vector, and back (rounded to T).
template <typename T>
HLM_DEVICE void f2_load(uint4 raw, F2 (&x)[8 / sizeof(T)]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (sizeof(T) == 4) {
    x[0] = f2(__uint_as_float(w[0]), __uint_as_float(w[1]));
    x[1] = f2(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = f2_unpack<T>(w[i]);
  }
}
template <typename T>
HLM_DEVICE uint4 f2_store(const F2 (&x)[8 / sizeof(T)]) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float a, b;
      f2_split(x[i], a, b);
      w[2 * i] = __float_as_uint(a);
      w[2 * i + 1] = __float_as_uint(b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      f2_split(x[i], a, b);
      w[i] = pack2<T>(a, b);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four codes of two pairs, packed low byte first.
HLM_DEVICE uint32_t quant_pack4(F2 x, F2 y, float inv) {
  float v0, v1, v2, v3;
  f2_split(x * f2(inv), v0, v1);
  f2_split(y * f2(inv), v2, v3);
  const uint32_t lo = __byte_perm(__float_as_uint(__fadd_rn(v0, 12582912.0f)), __float_as_uint(__fadd_rn(v1, 12582912.0f)), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(__fadd_rn(v2, 12582912.0f)), __float_as_uint(__fadd_rn(v3, 12582912.0f)), 0x0040);
  return inv == 0.0f ? 0u : __byte_perm(lo, hi, 0x5410);
}

// Four codes back as floats: each byte, offset by 128, becomes the low mantissa
// byte of 2^23, from which 2^23 + 128 is subtracted: exact.
HLM_DEVICE void codes_to_f2(uint32_t packed, F2& lo, F2& hi) {
  const uint32_t b = packed ^ 0x80808080u;
  const F2 off = f2(-8388736.0f);
  lo = f2(__uint_as_float(__byte_perm(b, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(b, 0x4b000000u, 0x7441))) + off;
  hi = f2(__uint_as_float(__byte_perm(b, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(b, 0x4b000000u, 0x7443))) + off;
}

// Largest magnitude among the elements of a 16-byte vector, as fp32 bits.  The
// 16-bit types compare as packed pairs of 15-bit integers: ordered like the
// magnitudes, infinities above finite values, NaNs above infinities.
template <typename T>
HLM_DEVICE uint32_t max16_packed(uint4 v);  // packed pair (16-bit types) or fp32 bits
template <>
HLM_DEVICE uint32_t max16_packed<float>(uint4 v) {
  constexpr uint32_t k = 0x7fffffffu;
  return max(max(v.x & k, v.y & k), max(v.z & k, v.w & k));
}
template <>
HLM_DEVICE uint32_t max16_packed<__nv_bfloat16>(uint4 v) {
  constexpr uint32_t k = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(v.x & k, v.y & k), __vmaxu2(v.z & k, v.w & k));
}
template <>
HLM_DEVICE uint32_t max16_packed<__half>(uint4 v) {
  return max16_packed<__nv_bfloat16>(v);
}
template <typename T>
HLM_DEVICE uint32_t max_packed(uint32_t a, uint32_t b) {
  return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b);
}
// fp32 magnitude bits of a packed maximum.
template <typename T>
HLM_DEVICE uint32_t unpack_max(uint32_t m);
template <>
HLM_DEVICE uint32_t unpack_max<float>(uint32_t m) {
  return m;
}
template <>
HLM_DEVICE uint32_t unpack_max<__nv_bfloat16>(uint32_t m) {
  return max(m & 0xffffu, m >> 16) << 16;
}
template <>
HLM_DEVICE uint32_t unpack_max<__half>(uint32_t m) {
  const uint16_t h = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
  return mag_bits(__half2float(__ushort_as_half(h)));
}

HLM_DEVICE uint32_t warp_max_u32(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

}  // namespace hlm
