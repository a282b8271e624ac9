// Reading rows of the 8-bit paged cache back (oscar_read_back): value = code 2^e,
// exact in every type it is written in.  A byte is read and two (or four) written for
// each value, so memory bounds it.  A thread takes 8 codes, so that a wave's loads and
// its 16-byte stores are each of consecutive addresses, and four of them at once.
// Measured: 24579 slots of a head of 256 8.9 us (38 MB, 4.2 TB/s: little more than a launch
// and a round trip), 65536 16.5 (101 MB, 6.1 TB/s), 32 users' 2K to 16K slots of 8 heads of
// 128 325 (1.8 GB, past the caches, 5.5 TB/s).
#include "quant_cache.h"
#include "quant_values.h"
#include "row_span.h"

#include <algorithm>

namespace oscar {
namespace {

constexpr int kReadThreads = 256;
constexpr int kReadItems = 4;              // of a thread
constexpr int64_t kLastCache = 256ll << 20;      // bytes

struct ReadArgs {
  const uint8_t* codes[2];                 // K, V
  const uint8_t* exponents;
  uint8_t* out[2];
  int64_t page[2], token[2], head[2];      // bytes
  int64_t out_token[2], out_head[2];
  const int64_t* slots;
  int64_t items, num_slots;
  int32_t block_size, num_heads;
  bool near;                               // slots fit 31 bits
  FastDiv by_token, by_head, by_block;     // items of a token, of a head
};

template <typename T, bool kOnce>
__global__ __launch_bounds__(kReadThreads) void read_kernel(ReadArgs a) {
  const int kv = (int)blockIdx.y;
  const int64_t first = (int64_t)blockIdx.x * (kReadThreads * kReadItems) + threadIdx.x;
  u32x2 codes[kReadItems];
  uint32_t exponent[kReadItems];
  uint8_t* to[kReadItems];
#pragma unroll
  for (int n = 0; n < kReadItems; ++n) {
    const int64_t item = first + n * kReadThreads;
    codes[n] = u32x2{};
    exponent[n] = 127;
    to[n] = nullptr;
    if (item >= a.items) continue;
    const uint32_t token = fast_div((uint32_t)item, a.by_token);
    const uint32_t in_token = (uint32_t)item - token * a.by_token.d;
    const uint32_t head = fast_div(in_token, a.by_head), piece = in_token - head * a.by_head.d;
    to[n] = a.out[kv] + (int64_t)token * a.out_token[kv] + (int64_t)head * a.out_head[kv] + 8 * sizeof(T) * piece;
    const int64_t slot = a.slots[token];
    if (slot < 0 || slot >= a.num_slots) continue;
    const int64_t page = a.near ? (int64_t)fast_div((uint32_t)slot, a.by_block) : slot / a.block_size;
    const int64_t in_page = slot - page * a.block_size;
    codes[n] = *reinterpret_cast<const u32x2*>(a.codes[kv] + page * a.page[kv] + in_page * a.token[kv] +
                                               (int64_t)head * a.head[kv] + 8 * piece);
    exponent[n] = a.exponents[2 * ((page * a.num_heads + head) * a.block_size + in_page) + kv];
  }
#pragma unroll
  for (int n = 0; n < kReadItems; ++n)
    if (to[n] != nullptr) store_values<T, kOnce>(to[n], codes[n], scale_of(exponent[n]));
}

template <typename T>
void launch_read(const ReadArgs& a, bool once, hipStream_t stream) {
  const dim3 grid((uint32_t)((a.items + kReadThreads * kReadItems - 1) / (kReadThreads * kReadItems)), 2);
  if (once) read_kernel<T, true><<<grid, kReadThreads, 0, stream>>>(a);
  else read_kernel<T, false><<<grid, kReadThreads, 0, stream>>>(a);
}

}  // namespace
}  // namespace oscar

extern "C" int oscar_read_back(const oscar_quant_cache* cache, const int64_t* slots, int64_t num_tokens,
                               const oscar_heads* key_out, const oscar_heads* value_out, int32_t dtype,
                               oscar_stream_t stream) {
  using namespace oscar;
  const int status = check_quant_cache(cache);
  if (status != kOk) return status;
  if (num_tokens < 0 || key_out == nullptr || value_out == nullptr || key_out->num_heads != cache->num_kv_heads ||
      value_out->num_heads != cache->num_kv_heads || (dtype != cache->dtype && dtype != OSCAR_FP32))
    return kErrInvalidArgument;
  if (num_tokens == 0) return kOk;
  if (slots == nullptr || key_out->data == nullptr || value_out->data == nullptr) return kErrInvalidArgument;
  const int64_t size = dtype == OSCAR_FP32 ? 4 : 2, row = size * cache->head_size;
  const int64_t per_token = (int64_t)cache->num_kv_heads * (cache->head_size / 8);
  ReadArgs a{};
  const oscar_heads* const out[2] = {key_out, value_out};
  const int64_t page[2] = {cache->k_stride_page, cache->v_stride_page};
  const int64_t token[2] = {cache->k_stride_token, cache->v_stride_token};
  const int64_t head[2] = {cache->k_stride_head, cache->v_stride_head};
  const uint8_t* const codes[2] = {static_cast<const uint8_t*>(cache->k), static_cast<const uint8_t*>(cache->v)};
  RowSpan spans[2];
  for (int i = 0; i < 2; ++i) {
    a.codes[i] = codes[i];
    a.page[i] = page[i], a.token[i] = token[i], a.head[i] = head[i];
    a.out[i] = static_cast<uint8_t*>(out[i]->data);
    a.out_token[i] = num_tokens > 1 ? out[i]->token_stride : 0;       // (of single rows they mean nothing)
    a.out_head[i] = cache->num_kv_heads > 1 ? out[i]->head_stride : 0;
    for (int64_t* const y : {&a.out_token[i], &a.out_head[i]}) {
      if (*y < 0 || *y > UINT32_MAX) return kErrUnsupportedGeometry;
      *y *= size;
    }
    if (((uintptr_t)a.out[i] | (uintptr_t)a.out_token[i] | (uintptr_t)a.out_head[i]) % 16)
      return kErrUnsupportedGeometry;
    spans[i] = RowSpan{(uint64_t)(uintptr_t)a.out[i], a.out_token[i], a.out_head[i], num_tokens, cache->num_kv_heads,
                       row};
  }
  if (!rows_apart(spans[0], spans[1])) return kErrOverlap;
  a.exponents = cache->exponents;
  a.num_slots = cache->num_pages * cache->block_size;
  a.near = a.num_slots <= INT32_MAX;
  a.block_size = cache->block_size;
  a.num_heads = cache->num_kv_heads;
  a.by_token = make_fast_div((uint32_t)per_token);
  a.by_head = make_fast_div((uint32_t)(cache->head_size / 8));
  a.by_block = make_fast_div((uint32_t)cache->block_size);
  const bool once = 2 * num_tokens * per_token * 8 * (1 + size) > kLastCache;
  // (a launch's items are counted in 31 bits)
  const int64_t most = (1ll << 30) / per_token;
  for (int64_t at = 0; at < num_tokens; at += most) {
    ReadArgs part = a;
    const int64_t tokens = std::min(most, num_tokens - at);
    part.slots = slots + at;
    part.items = tokens * per_token;
    for (int i = 0; i < 2; ++i) part.out[i] += at * a.out_token[i];
    if (dtype == OSCAR_BF16) launch_read<__bf16>(part, once, stream);
    else if (dtype == OSCAR_FP16) launch_read<_Float16>(part, once, stream);
    else launch_read<float>(part, once, stream);
  }
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}
