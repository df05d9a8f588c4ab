// Microscaled 4-bit floating point (OCP MX, "MXFP4"): 32 values of a row share
// one power of two (8-bit exponent, bias 127, 255 = NaN) and are held as e2m1
// codes (0 0.5 1 1.5 2 3 4 6 and a sign).
//
// A matrix [R, C] lies as K-slabs of 128 values of its rows: codes
// [mx_slabs(C)][mx_rows(R)][64] bytes (two values a byte, the lower in the
// lower half), scales [mx_slabs(C)][mx_rows(R)][4].  Rows are rounded up to 16
// and columns to 128; what is added holds zero codes and zero scales.
#pragma once
#include "common.h"

namespace sfp8 {

enum : int { kMxF32 = 0, kMxBf16 = 1, kMxF16 = 2 };

__host__ __device__ inline int64_t mx_slabs(int64_t C) { return (C + 127) / 128; }
__host__ __device__ inline int64_t mx_rows(int64_t R) { return (R + 15) / 16 * 16; }

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
// 16 bytes at any element's address: global memory takes them there in one access
typedef int mx_intx4_any __attribute__((ext_vector_type(4), aligned(2)));

// The scale of a block whose largest |value| has these fp32 bits: its exponent
// less that of the largest code (6 = 1.5 * 2^2), not below 2^-127; NaN where
// the block holds an infinity or a NaN.
SFP8_DEV uint32_t mx_scale_code(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23);
  return e == 255 ? 255u : (uint32_t)(e > 2 ? e - 2 : 0);
}
// ... as fp32 bits (2^-127 is subnormal there; the converters read the exponent field)
SFP8_DEV float mx_scale_value(uint32_t code) {
  return __uint_as_float(code == 255u ? 0x7fc00000u : code ? code << 23 : 0x00400000u);
}

// Eight values of one type as the kernels hold them, from memory at any
// element's address.
template <int DT>
struct Eight {
  uint32_t w[DT == kMxF32 ? 8 : 4];
};

template <int DT>
SFP8_DEV Eight<DT> load8(const void* p, int64_t i) {
  Eight<DT> v;
  if constexpr (DT == kMxF32) {
    typedef int any4 __attribute__((ext_vector_type(4), aligned(4)));
    const any4 a = *reinterpret_cast<const any4*>(reinterpret_cast<const float*>(p) + i);
    const any4 b = *reinterpret_cast<const any4*>(reinterpret_cast<const float*>(p) + i + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v.w[j] = (uint32_t)a[j], v.w[4 + j] = (uint32_t)b[j];
  } else {
    const mx_intx4_any a = *reinterpret_cast<const mx_intx4_any*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) v.w[j] = (uint32_t)a[j];
  }
  return v;
}

// The first n of eight values (n from 0 to 8), zeros behind them.
template <int DT>
SFP8_DEV Eight<DT> load8_upto(const void* p, int64_t i, int64_t n) {
  if (n >= 8) return load8<DT>(p, i);
  Eight<DT> v{};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j < n) {
      if constexpr (DT == kMxF32) v.w[j] = reinterpret_cast<const uint32_t*>(p)[i + j];
      else v.w[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i + j] << (16 * (j & 1));
    }
  }
  return v;
}

// The largest |value| of the eight as unsigned bits of its own type: their
// order is that of the values, NaN above all.
template <int DT>
SFP8_DEV uint32_t abs_max8(const Eight<DT>& v) {
  if constexpr (DT == kMxF32) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t a = v.w[j] & 0x7fffffffu;
      m = a > m ? a : m;
    }
    return m;
  } else {
    ushortx2 m = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(ushortx2, v.w[j] & 0x7fff7fffu));
    return m[0] > m[1] ? m[0] : m[1];
  }
}

template <int DT>
SFP8_DEV uint32_t abs_bits_to_f32(uint32_t m) {
  if constexpr (DT == kMxF32) return m;
  else if constexpr (DT == kMxBf16) return m << 16;
  else return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m));
}

// Two values (for 16-bit types one packed word, else two words) as the codes
// of byte SEL of `old`: value / scale rounded to nearest even, +-6 past that.
template <int DT, int SEL>
SFP8_DEV uint32_t cvt_codes(uint32_t old, uint32_t a, uint32_t b, float scale) {
  if constexpr (DT == kMxF32)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, __uint_as_float(a), __uint_as_float(b), scale, SEL);
  else if constexpr (DT == kMxBf16)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2_t, a), scale, SEL);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(halfx2, a), scale, SEL);
}

// The eight codes of eight values.
template <int DT>
SFP8_DEV uint32_t codes8(const Eight<DT>& v, float scale) {
  constexpr int n = DT == kMxF32 ? 2 : 1;  // words a pair
  uint32_t c = cvt_codes<DT, 0>(0u, v.w[0], v.w[n - 1], scale);
  c = cvt_codes<DT, 1>(c, v.w[n], v.w[2 * n - 1], scale);
  c = cvt_codes<DT, 2>(c, v.w[2 * n], v.w[3 * n - 1], scale);
  return cvt_codes<DT, 3>(c, v.w[3 * n], v.w[4 * n - 1], scale);
}

// Eight codes -> eight bf16 values times the scale (exact wherever bf16 holds them).
SFP8_DEV bf16x8 bf16_of_codes8(uint32_t c, float scale) {
  uint32_t w[4];
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
  w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
  w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
  return __builtin_bit_cast(bf16x8, intx4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]});
}

}  // namespace sfp8
