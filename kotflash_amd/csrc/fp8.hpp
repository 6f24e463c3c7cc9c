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

// Transposed read of an 8 x 16 block of bytes (ds_read_b64_tr_b8): inside each
// group of 16 lanes, lanes 2 r and 2 r + 1 address the halves of row r, and lane i
// receives column i. Checked on the device.
__device__ inline u32x2 lds_read_tr8(const uint8_t* p) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((KF_LDS i32x2*)(p)));
}

}  // namespace kf
