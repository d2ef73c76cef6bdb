// Microscaled 4-bit floating point on gfx950: blocks of 32 consecutive values share one scale byte s, and a value is
// e2m1(code) * 2^(s - 127).  e2m1 codes 0..7 are 0, 0.5, 1, 1.5, 2, 3, 4, 6, bit 3 is the sign; s = 255 makes the block NaN.
// Two codes a byte, the even element in the low nibble; rows are packed each on its own.
//
// The conversions are the hardware's (v_cvt_scalef32_pk_*): the scale operand is an fp32 of which only the exponent field
// counts, so s << 23 is the scale for every s, 0 (2^-127) and 255 (NaN) included.  Checked on the device: all 256 scales
// times all codes into bf16, f16 and fp32 are the exact product rounded once to nearest even (f16 overflows to
// infinity); fp32 -> code is x / 2^(s - 127) rounded to the nearest code, ties to the even one, saturated at 6.
#pragma once

#include "lds_stage.h"

namespace hk {

constexpr int kMxBlock = 32;

__device__ __forceinline__ float mx_scale(uint32_t s) { return __uint_as_float(s << 23); }

// Codes 2 SEL, 2 SEL + 1 of a dword of eight as two packed 16-bit values.
template <typename T, int SEL>
__device__ __forceinline__ uint32_t mx4_pair(uint32_t w, float s) {
  if constexpr (std::is_same<T, BF16>::value) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, SEL));
}
// Eight codes as eight 16-bit values: an operand fragment.
template <typename T>
__device__ __forceinline__ u32x4 mx4_unpack8(uint32_t w, float s) {
  return u32x4{mx4_pair<T, 0>(w, s), mx4_pair<T, 1>(w, s), mx4_pair<T, 2>(w, s), mx4_pair<T, 3>(w, s)};
}

// The scale byte of a block whose largest magnitude has these fp32 bits: floor(log2) - 2, so that the largest value falls
// into [4, 8) and is rounded or saturated to 4 or 6; 0 where that is below 2^-127 (all-zero blocks too), 255 for a block
// with an infinity or NaN.
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t abs_bits) {
  const uint32_t e = abs_bits >> 23;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

}  // namespace hk
