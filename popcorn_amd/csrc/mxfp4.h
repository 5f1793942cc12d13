// MXFP4 (OCP Microscaling): blocks of 32 values share a power of two, E8M0 byte
// e for 2^(e - 127) (255: NaN), and each value is an e2m1 code, sign in bit 3 and
// the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6 in the others. gfx950 converts two codes
// at a time, in either direction and with the scale applied, in one instruction;
// they read the scale's exponent field only.
#pragma once

#include "common.h"

namespace pk {
namespace mx {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The scale 2^(e - 127) as the conversions take it. The mantissa bit keeps byte 0
// from reading as a zero and 255 as an infinity.
__device__ __forceinline__ float scale_of(uint32_t e) { return __builtin_bit_cast(float, (e << 23) | 0x00400000u); }

// The scale byte of a block whose largest |y| has the bits `top`: floor(log2) - 2,
// so that the largest value lies in [4, 8) steps and what is over 6 saturates. 0 to
// 2^-124 take 2^-126. A block that holds a NaN or an Inf is NaN as a whole.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const uint32_t field = top >> 23;
  return field == 255u ? 255u : (field < 3u ? 1u : field - 2u);
}

// Eight values as their codes, the first in the lowest nibble; to nearest, ties to even.
__device__ __forceinline__ uint32_t encode8(const float (&y)[8], uint32_t e) {
  if (e == 255u) return 0u;
  const float s = scale_of(e);
  uint32_t r = 0u;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[0], y[1], s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2], y[3], s, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4], y[5], s, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6], y[7], s, 3);
  return r;
}

__device__ __forceinline__ void decode8(uint32_t codes, float s, float (&y)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
  y[0] = a.x, y[1] = a.y, y[2] = b.x, y[3] = b.y, y[4] = c.x, y[5] = c.y, y[6] = d.x, y[7] = d.y;
}

// The same as bf16 pairs (exact: three significant bits and bf16's exponents).
__device__ __forceinline__ uint4 decode8_bf16(uint32_t codes, float s) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0));
  r.y = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1));
  r.z = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2));
  r.w = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3));
  return r;
}

}  // namespace mx
}  // namespace pk
