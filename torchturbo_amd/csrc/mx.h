// Microscaling formats (OCP MX): groups of 32 elements share a power of two, kept as a byte c
// of value 2^(c - 127) (255: the group is NaN). Elements are E2M1 (two to a byte, the lower index in
// the low four bits) or E4M3.
//
// A group is quantised as the specification's conversion does: c = floor(log2 amax) - emax + 127
// with emax 2 (E2M1) or 8 (E4M3), elements v / 2^(c - 127) rounded to nearest even and kept within
// +-6 or +-448. A group of zeros has c = 0; NaN or infinity in a group gives c = 255.
#pragma once

#include "common.h"

constexpr int MX_GROUP = 32;

typedef __attribute__((ext_vector_type(2))) __bf16 mx_bf16x2;
typedef __attribute__((ext_vector_type(8))) float mx_f32x8;

// The byte of a group from its largest magnitude's bits (ordered as the values are, NaN on
// top).
template <int EMAX>
__device__ __forceinline__ uint32_t mx_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int e = (int)(amax_bits >> 23) - EMAX;  // exponent + 127 - EMAX; 0 for subnormals
  return e < 0 ? 0u : (uint32_t)e;
}

// 2^(c - 127) and its inverse as fp32 (c at most 252 from a finite fp32: both are representable,
// the first as a subnormal for c = 0).
__device__ __forceinline__ float mx_scale(uint32_t c) {
  return c == 0 ? 0x1p-127f : __uint_as_float(c == 255u ? 0x7fc00000u : c << 23);
}
__device__ __forceinline__ float mx_inverse(uint32_t c) { return __uint_as_float((254u - c) << 23); }

// Four values (already times the inverse scale) as E4M3 bytes, kept within +-448. The
// hardware's conversion rounds to nearest even.
__device__ __forceinline__ uint32_t mx_e4m3x4(float a, float b, float c, float d) {
  a = __builtin_amdgcn_fmed3f(a, -448.f, 448.f);
  b = __builtin_amdgcn_fmed3f(b, -448.f, 448.f);
  c = __builtin_amdgcn_fmed3f(c, -448.f, 448.f);
  d = __builtin_amdgcn_fmed3f(d, -448.f, 448.f);
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  return (uint32_t)v;
}

// Eight fp32 values as E2M1 codes in one word, of scale 2^(c - 127) given as fp32 (its exponent
// counts). The hardware rounds v / scale to nearest even and keeps it within +-6.
__device__ __forceinline__ uint32_t mx_e2m1x8(const float* v, float scale) {
  uint32_t q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], scale, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
}

// Eight E2M1 codes of scale byte c as bf16: exact, since a code has one fraction bit (as a
// subnormal where 2^(c - 127) is tiny). The conversion takes the scale's exponent alone, 0 as
// 2^-127, and gives NaN for 255.
__device__ __forceinline__ uint4 mx_bf16x8(uint32_t q, uint32_t c) {
  const float s = __uint_as_float(c << 23);
  const mx_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0);
  const mx_bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1);
  const mx_bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2);
  const mx_bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3);
  return uint4{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
               __builtin_bit_cast(uint32_t, d), __builtin_bit_cast(uint32_t, e)};
}

// Eight consecutive elements as fp32: one vector load of 16-bit elements or two of fp32
// (VEC: whole and 16-byte aligned), or up to `left` single ones, zeros behind them.
template <class T, bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const typename T::storage* p, int64_t left) {
  if constexpr (VEC) {
    typename T::storage s[8];
    *reinterpret_cast<uint4*>(s) = *reinterpret_cast<const uint4*>(p);
    if constexpr (sizeof(s[0]) == 4)
      *reinterpret_cast<uint4*>(s + 4) = *reinterpret_cast<const uint4*>(p + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = T::to_f32(s[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? T::to_f32(p[j]) : 0.f;
  }
}

template <class T, bool VEC>
__device__ __forceinline__ void store8(typename T::storage* p, const float (&v)[8], int64_t left) {
  if constexpr (VEC) {
    typename T::storage s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = T::from_f32(v[j]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(s);
    if constexpr (sizeof(s[0]) == 4)
      *reinterpret_cast<uint4*>(p + 4) = *reinterpret_cast<const uint4*>(s + 4);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = T::from_f32(v[j]);
  }
}

// The largest magnitude's bits of a group whose 32 elements four neighbouring lanes hold, eight each.
__device__ __forceinline__ uint32_t mx_amax4(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 1, TT_WAVE));
  return max(m, (uint32_t)__shfl_xor((int)m, 2, TT_WAVE));
}

// Eight elements of such a group as E4M3 codes; its byte goes to `byte`.
__device__ __forceinline__ uint2 mx_rows8(const float (&v)[8], uint32_t& byte) {
  byte = mx_byte<8>(mx_amax4(v));
  if (byte == 255u) return uint2{0x7f7f7f7fu, 0x7f7f7f7fu};
  const float s = mx_inverse(byte);
  return uint2{mx_e4m3x4(v[0] * s, v[1] * s, v[2] * s, v[3] * s),
               mx_e4m3x4(v[4] * s, v[5] * s, v[6] * s, v[7] * s)};
}
