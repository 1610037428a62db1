// Weights held as e2m1 codes with a ue8m0 scale byte per 32 of a row (the form smla_rotate_fp4 writes), as the
// operands of bf16 matrix products.  Every code times its scale is a bf16 number (magnitudes of 2 significant bits
// and any power of two, 2^-128 a subnormal; past the range infinity; byte 255 NaN), so a product of converted
// weights is the product of the weights: nothing is rounded before the fp32 accumulation.  The conversion is one
// instruction per two values (v_cvt_scalef32_pk_bf16_fp4), as fast as an addition (4 cycles a wave).
#pragma once

#include "smla_internal.h"

namespace smla_fp4 {

// the scale operand of a byte: the conversion takes the exponent field alone
__device__ inline float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// 8 codes (element 2i in the low half of byte i) times a scale, as 8 bf16
__device__ inline bf16x8_t to_bf16(uint32_t codes, float scale) {
  const u32x4_t v = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
  return as_bf16x8(v);
}

}  // namespace smla_fp4
