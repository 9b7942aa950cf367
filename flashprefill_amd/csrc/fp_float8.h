// 8-bit floats of the KV cache: e4m3 (4-bit significand, largest finite 448, no
// infinity) and e5m2 (3-bit significand, largest finite 57344). Every value of
// either is a bf16 and a fp16 value, so widening is exact.
#pragma once

#include "fp_attn_common.h"

namespace fp {

template <int F>
struct Float8;

template <>
struct Float8<FP_CACHE_E4M3> {
  static constexpr float kMax = 448.0f;
  template <bool HI>
  static __device__ __forceinline__ bf16x2 to_bf16(uint32_t w) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI);
  }
  template <bool HI>
  static __device__ __forceinline__ f16x2 to_f16(uint32_t w) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI);
  }
  template <bool HI>
  static __device__ __forceinline__ f32x2 to_f32(uint32_t w) {
    return __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), HI);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t from_f32(float a, float b, uint32_t old) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_cvt_pk_fp8_f32(a, b, static_cast<int>(old), HI));
  }
};

template <>
struct Float8<FP_CACHE_E5M2> {
  static constexpr float kMax = 57344.0f;
  template <bool HI>
  static __device__ __forceinline__ bf16x2 to_bf16(uint32_t w) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, HI);
  }
  template <bool HI>
  static __device__ __forceinline__ f16x2 to_f16(uint32_t w) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, HI);
  }
  template <bool HI>
  static __device__ __forceinline__ f32x2 to_f32(uint32_t w) {
    return __builtin_amdgcn_cvt_pk_f32_bf8(static_cast<int>(w), HI);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t from_f32(float a, float b, uint32_t old) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_cvt_pk_bf8_f32(a, b, static_cast<int>(old), HI));
  }
};

// bytes 0, 1 (or 2, 3) of w as a packed pair of the 16-bit type
template <typename T, int F, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  if constexpr (std::is_same_v<T, BF16>)
    return __builtin_bit_cast(uint32_t, Float8<F>::template to_bf16<HI>(w));
  else
    return __builtin_bit_cast(uint32_t, Float8<F>::template to_f16<HI>(w));
}
// 8 bytes as 8 values of the 16-bit type
template <typename T, int F>
__device__ __forceinline__ uint4 widen8(uint32_t lo, uint32_t hi) {
  return make_uint4(widen2<T, F, false>(lo), widen2<T, F, true>(lo), widen2<T, F, false>(hi),
                    widen2<T, F, true>(hi));
}

// scale of (KV head h) of a fixed scale; 1 for one per slot
__device__ __forceinline__ float fixed_scale(const CacheScales& s, int h) {
  return s.slot || s.p == nullptr ? 1.0f : s.p[h * s.sh];
}

}  // namespace fp
