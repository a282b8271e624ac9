// Causal attention of a step's new tokens over a plain (bf16 or fp16) paged
// cache that already holds their keys and values (oscar_chunk_attention).
#include "chunk_pieces.h"
#include "chunk_plan.h"

namespace oscar {
namespace {

// ---------------------------------------------------------------- kernels
// (LDS of fixed size: its place is then known when addresses are computed, which in
// the wide tiles' steps is one addition an operand less: D = 256, 9256 tokens over
// 15360 1190 -> 1130 us.)
template <typename T, int D>
__global__ __launch_bounds__(kThreads, narrow_wgs(D)) void narrow_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[narrow_lds(D, kTileKeys)];
  narrow_piece<T, D, kTileKeys>(a, a.pieces[blockIdx.x], smem);
}
template <typename T, int D>
__global__ __launch_bounds__(kThreads, kWideWgs) void wide_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[wide_lds(D)];
  wide_piece<T, D>(a, a.pieces[blockIdx.x], smem);
}
// A step with both.  Narrow pieces that fill the GPU come after the wide ones, where
// those leave room: reads at full rate leave the wide pieces' next stage late.  A few
// (plan_narrow) come first, and read for as long as the wide ones compute.  1024
// tokens over 4096 beside seven users' 4, D = 256: 71 us, the wide ones first 83.
// Measured: D = 128 119 to 133 us; the wide ones alone take 90 to 102, the narrow ones
// alone 38.
constexpr int kFewNarrow = kCus;
constexpr int mixed_lds(int d) { return std::max(narrow_lds(d, beside_keys(d)), wide_lds(d)); }
template <typename T, int D>
__global__ __launch_bounds__(kThreads, kWideWgs) void mixed_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[mixed_lds(D)];
  const int total = a.narrow + a.wide, lead = a.narrow <= kFewNarrow ? 0 : a.narrow;
  const int at = (int)blockIdx.x + lead, i = at < total ? at : at - total;
  if (i >= a.narrow) wide_piece<T, D>(a, a.pieces[i], smem);
  else narrow_piece<T, D, beside_keys(D)>(a, a.pieces[i], smem);
}

template <typename T, int D>
int launch(const ChunkArgs& a, const oscar_chunk_step& step, hipStream_t stream) {
  static_assert(kWideWgs * mixed_lds(D) <= 160 * 1024 && narrow_wgs(D) * narrow_lds(D, kTileKeys) <= 160 * 1024,
                "the workgroups of a CU must fit its 160 KiB of LDS");
  void (*const kernels[3])(ChunkArgs) = {&narrow_kernel<T, D>, &wide_kernel<T, D>, &mixed_kernel<T, D>};
  const int which = step.wide == 0 ? 0 : step.narrow == 0 ? 1 : 2;
  kernels[which]<<<step.narrow + step.wide, kThreads, 0, stream>>>(a);
  return launch_joins<T, D, false>(a, step, stream);
}

template <typename T>
int launch_sized(int d, const ChunkArgs& a, const oscar_chunk_step& step, hipStream_t stream) {
  if (d == 64) return launch<T, 64>(a, step, stream);
  if (d == 128) return launch<T, 128>(a, step, stream);
  return launch<T, 256>(a, step, stream);
}

int check_chunk_cache(const oscar_plain_cache* c) {
  const int status = check_plain_cache(c);
  if (status != kOk) return status;
  if (c->head_size != 64 && c->head_size != 128 && c->head_size != 256) return kErrUnsupportedHeadDim;
  const bool near = c->k_stride_page <= UINT32_MAX && c->v_stride_page <= UINT32_MAX;
  return c->block_size % 16 == 0 && near ? kOk : kErrUnsupportedGeometry;
}

}  // namespace
}  // namespace oscar

extern "C" int oscar_chunk_plan_shared(const int32_t* query_start_loc, const int32_t* seq_lens, int32_t num_requests,
                                       int32_t num_heads, int32_t window, const oscar_prefix* prefixes,
                                       int32_t num_prefixes, const oscar_plain_cache* cache, void* items,
                                       size_t items_size, oscar_chunk_step* step) {
  using namespace oscar;
  int status = check_chunk_cache(cache);
  if (status != kOk) return status;
  if (step == nullptr) return kErrInvalidArgument;
  int32_t pages = 0;
  status = check_step(query_start_loc, seq_lens, num_requests, num_heads, cache->num_kv_heads, window, cache->block_size,
                      &pages);
  if (status != kOk) return status;
  const int32_t group = num_heads / cache->num_kv_heads;
  try {
    std::vector<Prefix> shared;
    status = check_prefixes(prefixes, num_prefixes, query_start_loc, seq_lens, num_requests, group, window, shared);
    if (status != kOk) return status;
    Plan plan;
    make_plan(query_start_loc, seq_lens, num_requests, group, cache->num_kv_heads, plain_rule(cache->head_size), window,
              shared, plan);
    step->num_requests = num_requests;
    step->num_tokens = num_requests > 0 ? query_start_loc[num_requests] : 0;
    step->num_heads = num_heads;
    step->num_kv_heads = cache->num_kv_heads;
    step->head_size = cache->head_size;
    step->block_size = cache->block_size;
    step->window = std::min(window, kMostKeys);
    step->table_cols = pages;
    return pack_plan(plan, cache->head_size, items, items_size, step);
  } catch (...) {
    return kErrInvalidArgument;
  }
}

extern "C" int oscar_chunk_plan(const int32_t* query_start_loc, const int32_t* seq_lens, int32_t num_requests,
                                int32_t num_heads, int32_t window, const oscar_plain_cache* cache, void* items,
                                size_t items_size, oscar_chunk_step* step) {
  return oscar_chunk_plan_shared(query_start_loc, seq_lens, num_requests, num_heads, window, nullptr, 0, cache, items,
                                 items_size, step);
}

extern "C" int oscar_chunk_attention(const oscar_chunk_step* step, const void* items, const int32_t* block_table,
                                     int64_t block_table_stride, const oscar_plain_cache* cache,
                                     const oscar_heads* query, const oscar_heads* out, float scale, void* workspace,
                                     size_t workspace_size, oscar_stream_t stream) {
  using namespace oscar;
  const int status = check_chunk_cache(cache);
  if (status != kOk) return status;
  if (step == nullptr || query == nullptr || out == nullptr || query->num_heads != step->num_heads ||
      out->num_heads != step->num_heads || step->num_heads < 1 || step->num_heads % cache->num_kv_heads ||
      !(scale > 0.f) || !(scale <= 3.0e38f))
    return kErrInvalidArgument;
  if (step->num_kv_heads != cache->num_kv_heads || step->head_size != cache->head_size ||
      step->block_size != cache->block_size)
    return kErrInvalidArgument;
  if (step->narrow < 0 || step->wide < 0 || step->few_joins < 0 || step->joins < step->few_joins || step->parts < 0 ||
      step->join_rows < 0 || step->join_rows > kTileRows || (step->joins > step->few_joins && step->join_rows == 0))
    return kErrInvalidArgument;
  if (step->narrow + step->wide == 0) return kOk;
  ChunkArgs a{};
  const int bad = step_args(step, items, block_table, block_table_stride, query, out, scale, workspace, workspace_size,
                            step->workspace_size, a);
  if (bad != kOk) return bad;
  a.k = static_cast<const uint8_t*>(cache->k);
  a.v = static_cast<const uint8_t*>(cache->v);
  a.k_page = (uint32_t)cache->k_stride_page;
  a.v_page = (uint32_t)cache->v_stride_page;
  a.num_pages = cache->num_pages;
  a.k_token = (int32_t)cache->k_stride_token;
  a.v_token = (int32_t)cache->v_stride_token;
  a.k_head = (int32_t)cache->k_stride_head;
  a.v_head = (int32_t)cache->v_stride_head;
  return cache->dtype == OSCAR_BF16 ? launch_sized<__bf16>(cache->head_size, a, *step, stream)
                                    : launch_sized<_Float16>(cache->head_size, a, *step, stream);
}
