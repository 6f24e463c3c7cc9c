// e4m3 codes (OCP: 4 significant bits, largest 448, smallest step 2^-9, NaN but
// no infinity) of the 8-bit cache, on gfx950's conversions. Checked on the device
// for all codes, and exponents of the scale from -126 to 120: code * scale in
// one rounding, subnormal results included.
#pragma once
#include "kf_common.hpp"

namespace kf {

// Codes 0 and 1 of a word (HIGH: 2 and 3) times a power of two, as a pair of
// 16-bit elements.
template <typename T, bool HIGH>
__device__ inline uint32_t dequantise2(uint32_t codes, float scale) {
  if constexpr (std::is_same_v<T, _Float16>)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

}  // namespace kf
