// e4m3 codes and their scales, as every kernel makes and reads them.
//
// A block of 128 consecutive elements of a row shares a scale (weights: a block of 128 x 128).  Codes that are made here
// have as scale the least power of two that leaves no element beyond 448, e4m3's largest value: a division by it is exact,
// so a code is one rounding of its element (within 2^-4 of it, whatever the scale: e4m3 is a floating type) and two
// programs that quantise the same 16-bit values get the same codes, where 448 / max has an ulp of its own that decides
// ties.  Against max / 448 as scale the smallest elements of a block lose up to one bit of their subnormal codes.
// Scales that a caller brings may be any fp32 values.
#pragma once

#include "ccf_common.h"

namespace ccf {

typedef __bf16 bf16_t;
typedef int int8v __attribute__((ext_vector_type(8)));
typedef int int2v __attribute__((ext_vector_type(2)));

constexpr int kScaleBlock = 128;

__host__ __device__ inline int scale_blocks(int k) { return (k + kScaleBlock - 1) / kScaleBlock; }

// The power of two for a block whose largest magnitude is `top`, and its reciprocal; 448 = 1.75 * 2^8, so a mantissa beyond
// 1.75 takes the next exponent.  At least 2^-126, whose reciprocal is a normal number too.  Infinities and NaN leave a
// finite scale: their own codes are NaN, their neighbours' small.
__device__ __forceinline__ float block_scale(float top, float *inverse) {
  uint32_t e = (__float_as_uint(top) + 0x1fffffu) >> 23;
  e = e > 9u ? e : 9u;
  *inverse = __uint_as_float((262u - e) << 23);
  return __uint_as_float((e - 8u) << 23);
}

// Four codes of already scaled values.  The conversion rounds to nearest even and keeps NaN; beyond 448 only an infinity
// comes, which e4m3 does not have: NaN.
__device__ __forceinline__ int pack_fp8(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

}  // namespace ccf
