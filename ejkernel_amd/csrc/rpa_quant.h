// The 8-bit paged cache with a scale per block of tokens and head: addressing and code conversions.
//
//   kv_cache  [num_pages, 2 * num_kv_heads, page_size, head_dim] codes
//   kv_scales [num_pages, 2 * num_kv_heads, page_size / scale_block] fp32, element = code * scale
#pragma once

#include "rpa_device.h"
#include "rpa_host.h"
#include "rpa_tile_common.h"

namespace rpa {


// Types of the codes.
constexpr int kCodeI8 = 0, kCodeE4m3 = 1, kCodeE5m2 = 2;

// The largest code.
template <int kCode>
__device__ __forceinline__ constexpr float code_max() {
  return kCode == kCodeI8 ? 127.f : kCode == kCodeE4m3 ? 448.f : 57344.f;
}

// Two neighbouring codes of a word (elements 2 * kHi and 2 * kHi + 1) as a pair of bf16: exact for all three types
// (|int8| needs 7 bits, the floating types 4 and 3, and bf16's exponents cover theirs).
template <int kCode, bool kHi>
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t w) {
  if constexpr (kCode == kCodeE4m3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHi));
  } else if constexpr (kCode == kCodeE5m2) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, kHi));
  } else {
    // a float that holds an integer of 8 bits has zeros in its lower half: the pair is the two upper halves
    const float a = static_cast<float>(static_cast<int8_t>(w >> (kHi ? 16 : 0)));
    const float b = static_cast<float>(static_cast<int8_t>(w >> (kHi ? 24 : 8)));
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
}

template <int kCode>
__device__ __forceinline__ float code_to_f32(uint32_t w, int byte) {
  const uint32_t b = (w >> (8 * byte)) & 0xffu;
  if constexpr (kCode == kCodeI8) return static_cast<float>(static_cast<int8_t>(b));
  else if constexpr (kCode == kCodeE4m3) return __builtin_amdgcn_cvt_f32_fp8(b, 0);
  else return __builtin_amdgcn_cvt_f32_bf8(b, 0);
}

__device__ __forceinline__ int clamp_page(int page, int num_pages) { return min(max(page, 0), num_pages - 1); }

inline int code_of_dtype(int cache_dtype) {
  return cache_dtype == RPA_DTYPE_INT8 ? kCodeI8 : cache_dtype == RPA_DTYPE_FP8_E4M3 ? kCodeE4m3 : kCodeE5m2;
}

}  // namespace rpa
