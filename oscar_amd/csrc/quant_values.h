// Codes of the 8-bit cache as the values they stand for, by the conversions that take
// a power of two along (exact: four significant bits).
#pragma once

#include "oscar_common.h"

namespace oscar {

// 2^(byte - 127) (255, which no write leaves, would be an infinity).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(min(byte, 254u) << 23); }

typedef __bf16 bf16_pair __attribute__((ext_vector_type(2)));
typedef _Float16 half_pair __attribute__((ext_vector_type(2)));
typedef float float_pair __attribute__((ext_vector_type(2)));

template <typename T>
struct Pair;
template <>
struct Pair<__bf16> {
  typedef bf16_pair Type;
  template <bool kHigh>
  static __device__ __forceinline__ Type of(uint32_t codes, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, kHigh);
  }
};
template <>
struct Pair<_Float16> {
  typedef half_pair Type;
  template <bool kHigh>
  static __device__ __forceinline__ Type of(uint32_t codes, float scale) {
    return __builtin_bit_cast(Type, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, kHigh));
  }
};
template <>
struct Pair<float> {
  typedef float_pair Type;
  template <bool kHigh>
  static __device__ __forceinline__ Type of(uint32_t codes, float scale) {
    return __builtin_bit_cast(Type, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, kHigh));
  }
};

// Eight values of a row.
template <typename T>
struct Values8 {
  typename Pair<T>::Type p[4];
};
template <typename T>
__device__ __forceinline__ Values8<T> values8(u32x2 codes, float scale) {
  return Values8<T>{{Pair<T>::template of<false>(codes[0], scale), Pair<T>::template of<true>(codes[0], scale),
                     Pair<T>::template of<false>(codes[1], scale), Pair<T>::template of<true>(codes[1], scale)}};
}
// .. written; kOnce: past the caches.
template <typename T, bool kOnce>
__device__ __forceinline__ void store_values(uint8_t* to, u32x2 codes, float scale) {
  const Values8<T> x = values8<T>(codes, scale);
  u32x4 w[sizeof(T) / 2];
  __builtin_memcpy(w, &x, sizeof(w));
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    u32x4* at = reinterpret_cast<u32x4*>(to) + i;
    if constexpr (kOnce) __builtin_nontemporal_store(w[i], at);
    else *at = w[i];
  }
}

}  // namespace oscar
