// What the files of the 8-bit operators share: 8-bit floating point types and
// blocks of 128 values with one float32 scale each.
//
// A block's scale is a / L, with a its largest magnitude (2^-100 at least) and L
// the type's largest value; its codes are round(x * (L / a)), each operation a
// float32 one, rounded to nearest.  A block that holds a NaN or an infinity has a
// NaN for its scale and for all of its codes.
#pragma once

#include "common.h"
#include "../../include/tilec.h"

namespace tilec {

constexpr int kGroup = 128;  // values of a row under one scale
constexpr float kSmallest = 0x1p-100f;

inline bool is_fp8(int32_t dtype) { return dtype == TILEC_F8E4M3 || dtype == TILEC_F8E5M2; }

__host__ __device__ constexpr float fp8_largest(bool e5m2) { return e5m2 ? 57344.f : 448.f; }

// The scale and its inverse of a block, from the bits of its largest magnitude
// (as integers they order like the magnitudes, infinities and NaNs above all).
__device__ __forceinline__ void block_scale(uint32_t top, float largest, float& scale, float& inverse) {
  const float a = top < 0x7f800000u ? fmaxf(__uint_as_float(top), kSmallest) : __uint_as_float(0x7fc00000u);
  scale = a / largest;
  inverse = largest / a;
}

// Four codes, the first in the lowest byte.
__device__ __forceinline__ uint32_t to_fp8(float a, float b, float c, float d, bool e5m2) {
  int v;
  if (e5m2) {
    v = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
    v = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, v, true);
  } else {
    v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  }
  return (uint32_t)v;
}

// The bits of a word of four codes that are those of the `left` (any number) of a row.
__device__ __forceinline__ uint32_t code_bits(int left) {
  return left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
}

}  // namespace tilec
