// Blocks of 8-bit codes (gfx950): K or V of one page and kv head as OCP e4m3 codes
// and the exponent of their scale, value = code * 2^exp.
//
// The exponent of a block is the smallest e with max |x| <= 448 * 2^e (448: e4m3's
// largest), held to kMinExp .. kMaxExp.  A power of two, because e4m3 is itself a
// floating format: any scale that keeps the largest value in range leaves the others
// their four significant bits, and a block whose exponent has to grow for a later
// token moves its older codes by an exponent, which is exact but for those that
// become subnormal.  At kMinExp the smallest code, 2^-9, stands for 2^-24, so every
// value is an fp16 number: nothing is lost by going from codes to fp16 (one
// instruction per two, scale included).  At kMaxExp codes end at 240 (kLargest):
// 256 * 2^8 would be fp16's infinity.  Values that are not finite are held as NaN,
// and count nothing in the maximum.
#pragma once

#include "device.hpp"

namespace aoakv {

constexpr int kMinExp = -15, kMaxExp = 8;
constexpr float kLargest = 61440.f;
typedef short short2v __attribute__((ext_vector_type(2)));

// 2^e of an exponent as the tables hold it (whatever they hold: in range)
__device__ inline float exp_scale(int e) {
  e = e < kMinExp ? kMinExp : e > kMaxExp ? kMaxExp : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// the exponent of a block whose largest finite |x| has these fp16 bits
__device__ inline int block_exp(uint32_t top) {
  const uint32_t u = __float_as_uint((float)__builtin_bit_cast(f16, (uint16_t)top));
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // 448 = 1.75 2^8
  return e < kMinExp ? kMinExp : e > kMaxExp ? kMaxExp : e;
}

// 4 codes as fp16 values, and 8
__device__ inline void decode4(uint32_t codes, float scale, half2v (&x)[2]) {
  x[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false);
  x[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true);
}
__device__ inline H8 decode8(uint2 codes, float scale) {
  half2v x[4];
  x[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes.x, scale, false);
  x[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes.x, scale, true);
  x[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes.y, scale, false);
  x[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes.y, scale, true);
  return __builtin_bit_cast(H8, x);
}

// 8 fp16 values as codes at the scale 2^e (|x| <= 448 * 2^e where finite; one
// rounding, to nearest even; inf and NaN become NaN)
__device__ inline uint2 encode8(const H8& v, int e) {
  const float scale = exp_scale(e);
  H8 x = v;
  if (e == kMaxExp) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const float f = (float)x.v[j];
      if (__builtin_isfinite(f)) x.v[j] = (f16)fminf(fmaxf(f, -kLargest), kLargest);
    }
  }
  short2v lo = {0, 0}, hi = {0, 0};
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(lo, half_pair(x, 0), scale, false);
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(lo, half_pair(x, 1), scale, true);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(hi, half_pair(x, 2), scale, false);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(hi, half_pair(x, 3), scale, true);
  return uint2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

// The larger of two pairs of |x| (fp16 bits order as whole numbers do), over 8 values.
__device__ inline uint32_t pair_top(const H8& v, uint32_t top) {
  typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
  const uint4 u = __builtin_bit_cast(uint4, v);
  ushort2v t = __builtin_bit_cast(ushort2v, top);
  t = __builtin_elementwise_max(t, __builtin_bit_cast(ushort2v, u.x & 0x7FFF7FFFu));
  t = __builtin_elementwise_max(t, __builtin_bit_cast(ushort2v, u.y & 0x7FFF7FFFu));
  t = __builtin_elementwise_max(t, __builtin_bit_cast(ushort2v, u.z & 0x7FFF7FFFu));
  t = __builtin_elementwise_max(t, __builtin_bit_cast(ushort2v, u.w & 0x7FFF7FFFu));
  return __builtin_bit_cast(uint32_t, t);
}
// The largest |x| among 8 values and `top` (fp16 bits): what is not finite counts 0.
__device__ inline uint32_t finite_top(const H8& v, uint32_t top) {
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const uint32_t y = __builtin_bit_cast(uint16_t, v.v[j]) & 0x7FFFu;
    if (y < 0x7C00u && y > top) top = y;
  }
  return top;
}

}  // namespace aoakv
