// The 8-bit paged cache (struct oscar_quant_cache): checks of its geometry, and how a
// row of values becomes codes and one power of two, and back.
//
// A code is an e4m3 number (sign, 4 bits of exponent, 3 of mantissa; largest 448, no
// infinities), a value code * 2^e, e one for a token and head.  The power is the
// smallest with which the row's largest finite magnitude is at most 448 2^e: being
// floating, the codes lose nothing by its steps of two.  Such values are exact in
// bf16, and in fp16 within its exponents, so whoever reads them adds no rounding.
#pragma once

#include "oscar_common.h"
#include "../../include/oscar_amd.h"

namespace oscar {

// e of bf16 rows: 2^-80 to 2^100, with which a sum of weights over 2^e, which the attention
// keeps, stays within fp32.  Of fp16 ones: 2^-9 2^-15 is its own smallest step, and 240 2^8
// the largest value below 65504, so that codes of the greatest power end at 240 (of bf16
// ones too: past 240 2^100 = 2^107.9).
struct ExponentRange {
  int low, high;
};
constexpr ExponentRange exponent_range(int dtype) {
  return dtype == OSCAR_FP16 ? ExponentRange{-15, 8} : ExponentRange{-80, 100};
}

__device__ __forceinline__ float power_of_two(int n) { return __int_as_float((n + 127) << 23); }   // -126 .. 127

__device__ __forceinline__ float finite_size(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.f;
}
__device__ __forceinline__ int row_exponent(float top, int low, int high) {
  const uint32_t bits = __float_as_uint(top);
  const int e = (int)(bits >> 23) - 127 - ((bits & 0x7FFFFFu) > 0x600000u ? 7 : 8);      // 448 = 1.75 * 2^8
  return min(max(e, low), high);
}
// Before rounding: within the codes, and what is not finite is NaN.
__device__ __forceinline__ float code_value(float x, float scale, float most) {
  const float y = x * scale;
  return fabsf(x) < __builtin_inff() ? fminf(fmaxf(y, -most), most) : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t codes4(const float* x, float scale, float most) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(code_value(x[0], scale, most), code_value(x[1], scale, most), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(code_value(x[2], scale, most), code_value(x[3], scale, most), w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ uint32_t code1(float x, float scale, float most) {
  const float y = code_value(x, scale, most);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xFFu;
}

// Codes and rows are 16-byte loads at 16-byte strides; inside a page offsets are
// 32-bit, so a page spans less than 2 GiB.
inline int check_quant_cache(const oscar_quant_cache* c) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->exponents == nullptr || c->num_pages < 1 ||
      c->block_size < 1 || c->num_kv_heads < 1 || (c->dtype != OSCAR_BF16 && c->dtype != OSCAR_FP16))
    return kErrInvalidArgument;
  if (c->head_size < 16 || c->head_size > 256 || c->head_size % 16) return kErrUnsupportedHeadDim;
  const int64_t row = c->head_size;
  const int64_t strides[2][3] = {{c->k_stride_page, c->k_stride_token, c->k_stride_head},
                                 {c->v_stride_page, c->v_stride_token, c->v_stride_head}};
  for (const auto& s : strides) {
    for (const int64_t x : s)
      if (x < row || x % 16) return kErrUnsupportedGeometry;
    if (s[1] >= INT32_MAX || s[2] >= INT32_MAX) return kErrUnsupportedGeometry;      // (the sums below fit 64 bits)
    const int64_t tokens = (int64_t)(c->block_size - 1) * s[1] + row, heads = (int64_t)(c->num_kv_heads - 1) * s[2] + row;
    const int64_t span = tokens + heads - row;
    if (span > INT32_MAX || (c->num_pages > 1 && s[0] < span)) return kErrUnsupportedGeometry;
    if (c->block_size > 1 && c->num_kv_heads > 1 && (s[1] < s[2] ? s[2] < tokens : s[1] < heads))
      return kErrUnsupportedGeometry;
  }
  if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->exponents) % 16) return kErrUnsupportedGeometry;
  return kOk;
}

}  // namespace oscar
