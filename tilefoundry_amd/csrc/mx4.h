// What the microscaled kernels share: the packed layout's sizes and the exact
// conversion of e2m1 codes to bf16 operands.
//
// Packed weights: blocks of 16 rows x 128 k, 1 KiB each, lane l's 16 bytes being
// the 32 codes of row l % 16 from k = 32 (l / 16) on.  That is one operand of the
// scaled 16x16x128 matrix instruction as it lies, with one scale a lane; and, its
// four dwords taken in turn, four operands of the bf16 16x16x32 instruction whose
// k runs over 32 (l / 16) + 8 step + 0 .. 7 (a product's k may be taken in any
// order that both operands share).  The scales follow all codes: lane l's four
// bytes for four consecutive blocks make one dword.
#pragma once

#include "panel.h"

namespace tfd {

constexpr int kMx4K = 128;   // k of a block
__host__ __device__ inline int mx4_blocks(int K) { return (K + kMx4K - 1) / kMx4K; }
__host__ __device__ inline int mx4_scale_groups(int kb) { return (kb + 3) / 4; }

// The scale byte as the f32 that the scaled conversions take: they read the
// exponent field alone, so 0 is 2^-127 and 255 is NaN.
__device__ __forceinline__ float mx4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes times a power of two, exact in bf16.
__device__ __forceinline__ u32x4 fp4x8_to_bf16(uint32_t q, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
  return u32x4{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
               __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)};
}

}  // namespace tfd
