// Checks of a plain paged cache's geometry (struct oscar_plain_cache), shared
// by its write and its reads.
#pragma once

#include "oscar_common.h"
#include "../../include/oscar_amd.h"

namespace oscar {

// Rows are 16-byte loads at 16-byte strides; inside a page offsets are 32-bit,
// so a page spans less than 2 GiB.
inline int check_plain_cache(const oscar_plain_cache* c) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->num_pages < 1 || c->block_size < 1 ||
      c->num_kv_heads < 1 || (c->dtype != OSCAR_BF16 && c->dtype != OSCAR_FP16))
    return kErrInvalidArgument;
  if (c->head_size < 8 || c->head_size > 256 || c->head_size % 8) return kErrUnsupportedHeadDim;
  const int64_t row = 2 * (int64_t)c->head_size;
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
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16) return kErrUnsupportedGeometry;
  return kOk;
}

}  // namespace oscar
