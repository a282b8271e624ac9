// Position rotation of queries and keys (oscar_rotate_positions), and the write
// of a step's keys and values to a plain paged cache with that rotation on the
// way (oscar_append_rotated).
//
// A head's pair (x1, x2) becomes (x1 c - x2 s, x2 c + x1 s) with the cosine and
// sine of its token's position on the pair's axis: fp32 arithmetic, one rounding
// to the rows' type.  Every value is read once and written once, so memory
// bounds the kernel (three flops a value), and for a few tokens its latency.
//
// A workgroup takes a block of tokens.  It collects their cosines and sines in
// LDS (each table entry read once for all heads, each pair from its own axis'
// row).  The rows' values go by in five jobs, one after the other: the turning
// parts of queries and keys (a thread to kVec pairs), their parts past
// rotary_dim and the values (a thread to kVec values).  A job's strides and
// divisors are the same for all lanes, so they stay in scalar registers (with all
// kinds of rows in one sequence of pieces each lane looked its own up: a write of
// 65536 tokens 176 us instead of 119).  Every job's first round of loads goes out
// before the cosines are collected.
//
// Measured: 30843 tokens of 32 + 8 heads of 128 (fp16, adjacent pairs) 112 us,
// 5.8 TB/s; a write of 65536 tokens of 6 + 1 + 1 heads of 256 105 us, 5.2 TB/s (a copy
// of 1 GiB moves 5.1 TB/s); 9256 of 6 + 1 heads of 256 (64 features turn, three axes)
// 13.4 us, 5.2 TB/s: called again and again, these 69 MB stay in the last-level cache,
// where a copy of as many bytes moves 6.6.  One token takes 5 us: positions, table and
// rows, a memory round trip each.
#include "plain_cache.h"
#include "row_span.h"

#include <type_traits>

namespace oscar {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxTokens = 16;             // of a workgroup
constexpr int kMaxRotary = 256;
constexpr int64_t kLastCache = 256ll << 20;      // bytes

// What a launch does with one part of one kind of rows: `pieces` a head, from
// feature `first` on.
struct Job {
  const uint8_t* src;
  uint8_t* dst;            // rows of its own, or a cache
  uint32_t src_token, src_head, dst_token, dst_head;   // bytes; in a cache dst_token is not used
  int32_t a_token;         // pieces of a token: heads x pieces
  int32_t pieces, first;
  FastDiv by_token, by_head;
};
constexpr int kJobs = 5;                   // turned: queries, keys; copied: queries, keys, values
constexpr bool turns(int job) { return job < 2; }

struct RotArgs {
  Job job[kJobs];
  const float* table;
  const int64_t* positions;
  int64_t axis_stride, table_rows, tokens;
  uint64_t pair_axis[4];
  const int64_t* slots;    // null: keys have rows of their own
  int64_t num_slots, k_page, k_token, v_page, v_token;
  int32_t block_size, block_shift;         // shift: log2, or -1
  int32_t axes, half;      // half: rotary_dim / 2
  int32_t block_tokens;
  float sign;              // of the sines
  FastDiv by_half;
};

template <typename T, int kVec>
struct Piece {
  typedef T Row __attribute__((ext_vector_type(kVec)));
};
template <typename T>
struct Piece<T, 1> {
  typedef T Row;
};

// Rows past the caches, where they would only push out what is read again.
template <bool kOnce, typename Row>
__device__ __forceinline__ Row load_row(const Row* x) {
  if constexpr (kOnce) return __builtin_nontemporal_load(x);
  else return *x;
}
template <bool kOnce, typename Row>
__device__ __forceinline__ void store_row(Row* y, Row x) {
  if constexpr (kOnce) __builtin_nontemporal_store(x, y);
  else *y = x;
}

// kVec values to a load: 16 bytes where rows, strides and pairs allow, else one
// value (a model's head size and projection decide, not the caller).
template <typename T, int kVec, bool kAdjacent, bool kOnce>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs a) {
  typedef typename Piece<T, kVec>::Row Row;
  __shared__ __attribute__((aligned(16))) float cs[kMaxTokens * kMaxRotary];   // [token][cos | sin]
  __shared__ int64_t at_k[kMaxTokens], at_v[kMaxTokens];                       // byte offset of the slot, -1: none
  __shared__ int live[kMaxTokens];
  const int tid = (int)threadIdx.x;
  const int64_t tok0 = (int64_t)blockIdx.x * a.block_tokens;
  const int tokens = (int)min((int64_t)a.block_tokens, a.tokens - tok0);
  constexpr int kPairs = kAdjacent && kVec > 1 ? kVec / 2 : kVec;     // of a turning piece
  constexpr int kSpan = kAdjacent && kVec == 1 ? 2 : kVec;            // features from one turning piece to the next
  const int width = 2 * a.half;

  struct Work {
    Row a, b;
    int token, head, feature, pair;
  };
  auto fetch = [&](auto tag, int idx, Work& w) {
    constexpr int kJob = decltype(tag)::value;
    const Job& j = a.job[kJob];
    w.token = (int)fast_div((uint32_t)idx, j.by_token);
    const int p = idx - w.token * j.a_token;
    w.head = (int)fast_div((uint32_t)p, j.by_head);
    const int piece = p - w.head * j.pieces;
    w.feature = j.first + piece * (turns(kJob) ? kSpan : kVec);
    w.pair = piece * kPairs;
    const T* x = reinterpret_cast<const T*>(j.src + tok0 * j.src_token + (uint64_t)(uint32_t)w.token * j.src_token +
                                            (uint64_t)(uint32_t)w.head * j.src_head) + w.feature;
    w.a = load_row<kOnce>(reinterpret_cast<const Row*>(x));
    if constexpr (turns(kJob) && !kAdjacent) w.b = load_row<kOnce>(reinterpret_cast<const Row*>(x + a.half));
    else if constexpr (turns(kJob) && kVec == 1) w.b = load_row<kOnce>(reinterpret_cast<const Row*>(x + 1));
  };
  auto finish = [&](auto tag, const Work& w) {
    constexpr int kJob = decltype(tag)::value;
    const Job& j = a.job[kJob];
    if (live[w.token] == 0) return;
    uint8_t* dst = j.dst + (uint64_t)(uint32_t)w.head * j.dst_head;
    constexpr bool kValue = kJob == 4, kKey = kJob == 1 || kJob == 3;
    if ((kKey && a.slots != nullptr) || kValue) {
      const int64_t at = kKey ? at_k[w.token] : at_v[w.token];
      if (at < 0) return;
      dst += at;
    } else {
      dst += tok0 * j.dst_token + (uint64_t)(uint32_t)w.token * j.dst_token;
    }
    T* y = reinterpret_cast<T*>(dst) + w.feature;
    if constexpr (!turns(kJob)) {
      store_row<kOnce>(reinterpret_cast<Row*>(y), w.a);
    } else {
      const float* c = cs + w.token * width + w.pair;
      const float* sn = c + a.half;
      if constexpr (kVec == 1) {
        const float x1 = (float)w.a, x2 = (float)w.b;
        y[0] = (T)(x1 * c[0] - x2 * sn[0]);
        y[kAdjacent ? 1 : a.half] = (T)(x2 * c[0] + x1 * sn[0]);
      } else if constexpr (kAdjacent) {
        Row o;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const float x1 = (float)w.a[2 * i], x2 = (float)w.a[2 * i + 1];
          o[2 * i] = (T)(x1 * c[i] - x2 * sn[i]);
          o[2 * i + 1] = (T)(x2 * c[i] + x1 * sn[i]);
        }
        store_row<kOnce>(reinterpret_cast<Row*>(y), o);
      } else {
        Row o1, o2;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float x1 = (float)w.a[i], x2 = (float)w.b[i];
          o1[i] = (T)(x1 * c[i] - x2 * sn[i]);
          o2[i] = (T)(x2 * c[i] + x1 * sn[i]);
        }
        store_row<kOnce>(reinterpret_cast<Row*>(y), o1);
        store_row<kOnce>(reinterpret_cast<Row*>(y + a.half), o2);
      }
    }
  };
  auto each_job = [&](auto&& f) {
    f(std::integral_constant<int, 0>{});
    f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 3>{});
    f(std::integral_constant<int, 4>{});
  };

  Work w0[kJobs];
  each_job([&](auto tag) {
    constexpr int kJob = decltype(tag)::value;
    if (tid < tokens * a.job[kJob].a_token) fetch(tag, tid, w0[kJob]);
  });

  // The tokens' cosines and sines, slots and whether their positions exist.
  for (int i = tid; i < tokens * a.half; i += kRotThreads) {
    const int t = (int)fast_div((uint32_t)i, a.by_half);
    const int j = i - t * a.half;
    const int axis = (int)(a.pair_axis[j >> 5] >> (2 * (j & 31))) & 3;
    const int64_t pos = a.positions[axis * a.axis_stride + tok0 + t];
    const bool in = pos >= 0 && pos < a.table_rows;
    const float* row = a.table + (in ? pos : 0) * width;
    cs[t * width + j] = row[j];
    cs[t * width + a.half + j] = row[a.half + j] * a.sign;
  }
  if (tid < tokens) {
    bool in = true;
    for (int x = 0; x < a.axes; ++x) {
      const int64_t pos = a.positions[x * a.axis_stride + tok0 + tid];
      in = in && pos >= 0 && pos < a.table_rows;
    }
    live[tid] = in;
    if (a.slots != nullptr) {
      const int64_t slot = a.slots[tok0 + tid];
      const bool write = slot >= 0 && slot < a.num_slots;
      const int64_t s = write ? slot : 0;
      const int64_t page = a.block_shift >= 0 ? s >> a.block_shift : s / a.block_size;
      const int64_t in_page = s - page * a.block_size;
      at_k[tid] = write ? page * a.k_page + in_page * a.k_token : -1;
      at_v[tid] = write ? page * a.v_page + in_page * a.v_token : -1;
    }
  }
  __syncthreads();

  each_job([&](auto tag) {
    constexpr int kJob = decltype(tag)::value;
    const int count = tokens * a.job[kJob].a_token;
    if (tid < count) finish(tag, w0[kJob]);
    for (int idx = tid + kRotThreads; idx < count; idx += 2 * kRotThreads) {
      Work u, v;
      const bool two = idx + kRotThreads < count;
      fetch(tag, idx, u);
      if (two) fetch(tag, idx + kRotThreads, v);
      finish(tag, u);
      if (two) finish(tag, v);
    }
  });
}

template <typename T, int kVec, bool kOnce>
void launch_kernel(const RotArgs& a, bool adjacent, hipStream_t stream) {
  const dim3 grid((uint32_t)((a.tokens + a.block_tokens - 1) / a.block_tokens));
  if (adjacent) rotary_kernel<T, kVec, true, kOnce><<<grid, kRotThreads, 0, stream>>>(a);
  else rotary_kernel<T, kVec, false, kOnce><<<grid, kRotThreads, 0, stream>>>(a);
}
template <typename T>
void launch_typed(const RotArgs& a, bool vec, bool once, bool adjacent, hipStream_t stream) {
  constexpr int kVec = 16 / (int)sizeof(T);
  if (!vec) launch_kernel<T, 1, false>(a, adjacent, stream);
  else if (once) launch_kernel<T, kVec, true>(a, adjacent, stream);
  else launch_kernel<T, kVec, false>(a, adjacent, stream);
}

int dtype_size(int32_t dtype) { return dtype == OSCAR_FP32 ? 4 : 2; }

// One kind of rows: where they come from and go to (out null: a cache).
struct Rows {
  const uint8_t* src;
  uint8_t* dst;
  int64_t src_token, src_head, dst_token, dst_head;    // bytes
  int32_t heads;
};

RowSpan source(const Rows& s, int64_t tokens, int64_t row) {
  return RowSpan{(uint64_t)(uintptr_t)s.src, s.src_token, s.src_head, tokens, s.heads, row};
}
RowSpan target(const Rows& s, int64_t tokens, int64_t row) {
  return RowSpan{(uint64_t)(uintptr_t)s.dst, s.dst_token, s.dst_head, tokens, s.heads, row};
}

bool fits16(const void* p, int64_t token_bytes, int64_t head_bytes) {
  return ((uintptr_t)p | (uintptr_t)token_bytes | (uintptr_t)head_bytes) % 16 == 0;
}

// (Strides between rows of which there is one mean nothing.)
int make_rows(Rows& s, const oscar_heads* in, const oscar_heads* out, int64_t tokens, int size, bool& vec) {
  if (in == nullptr || in->num_heads == 0) return kOk;
  if (in->data == nullptr || in->num_heads < 0 || in->num_heads > (1 << 16)) return kErrInvalidArgument;
  s.src = static_cast<const uint8_t*>(in->data);
  s.src_token = tokens > 1 ? in->token_stride * size : 0;
  s.src_head = in->num_heads > 1 ? in->head_stride * size : 0;
  s.heads = in->num_heads;
  vec = vec && fits16(s.src, s.src_token, s.src_head);
  if (out != nullptr) {
    if (out->data == nullptr || out->num_heads != in->num_heads) return kErrInvalidArgument;
    s.dst = static_cast<uint8_t*>(out->data);
    s.dst_token = tokens > 1 ? out->token_stride * size : 0;
    s.dst_head = out->num_heads > 1 ? out->head_stride * size : 0;
    vec = vec && fits16(s.dst, s.dst_token, s.dst_head);
  }
  for (const int64_t x : {s.src_token, s.src_head, s.dst_token, s.dst_head})
    if (x < 0 || x > UINT32_MAX) return kErrUnsupportedGeometry;
  return kOk;
}

int run(const oscar_rotary* r, const int64_t* positions, int64_t axis_stride, int64_t tokens, const oscar_heads* query,
        const oscar_heads* query_out, const oscar_heads* key, const oscar_heads* key_out, const oscar_heads* value,
        const oscar_plain_cache* cache, const int64_t* slots, int32_t head_size, int32_t dtype, int32_t inverse,
        hipStream_t stream) {
  if (tokens < 0 || r == nullptr || r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > kMaxRotary ||
      r->axes < 1 || r->axes > 4 || r->positions < 1 || dtype < OSCAR_BF16 || dtype > OSCAR_FP32)
    return kErrInvalidArgument;
  if (head_size < r->rotary_dim || head_size % 2 || head_size > 256) return kErrUnsupportedHeadDim;
  for (int j = 0; j < r->rotary_dim / 2; ++j)
    if ((int)((r->pair_axis[j >> 5] >> (2 * (j & 31))) & 3) >= r->axes) return kErrInvalidArgument;
  if (tokens == 0) return kOk;
  if (r->table == nullptr || positions == nullptr) return kErrInvalidArgument;
  const int size = dtype_size(dtype);
  RotArgs a{};
  bool vec = true;
  Rows rows[3] = {};
  const oscar_heads* const in[3] = {query, key, value};
  const oscar_heads* const out[3] = {query_out, key_out, nullptr};
  for (int i = 0; i < 3; ++i) {
    const int status = make_rows(rows[i], in[i], out[i], tokens, size, vec);
    if (status != kOk) return status;
  }
  // An output that is its input is read and written row by row by one thread; of any
  // other rows that it shares memory with, some would be read after they are written.
  const int64_t row = (int64_t)head_size * size;
  for (int i = 0; i < 2; ++i) {
    if (out[i] == nullptr) continue;
    const RowSpan to = target(rows[i], tokens, row);
    for (int j = 0; j < 3; ++j) {
      const RowSpan from = source(rows[j], tokens, row);
      if (!(i == j && same_rows(to, from)) && !rows_apart(to, from)) return kErrOverlap;
    }
    if (i == 0 && out[1] != nullptr && !rows_apart(to, target(rows[1], tokens, row))) return kErrOverlap;
  }
  if (cache != nullptr) {
    rows[1].dst = static_cast<uint8_t*>(cache->k);
    rows[1].dst_head = cache->k_stride_head;
    rows[2].dst = static_cast<uint8_t*>(cache->v);
    rows[2].dst_head = cache->v_stride_head;
    a.slots = slots;
    a.num_slots = cache->num_pages * cache->block_size;
    a.k_page = cache->k_stride_page;
    a.k_token = cache->k_stride_token;
    a.v_page = cache->v_stride_page;
    a.v_token = cache->v_stride_token;
    a.block_size = cache->block_size;
    a.block_shift = -1;
    for (int s = 0; s < 31; ++s)
      if (cache->block_size == (1 << s)) a.block_shift = s;
  }
  // A 16-byte piece of a turning row: 16 bytes of both partners' halves, or of
  // adjacent pairs.
  const int wide = 16 / size;
  vec = vec && head_size % wide == 0 && (r->adjacent ? r->rotary_dim : r->rotary_dim / 2) % wide == 0;
  const int step = vec ? wide : 1;
  int64_t work = 0, read = 0;               // pieces and bytes of a token
  for (int i = 0; i < kJobs; ++i) {
    const Rows& s = rows[turns(i) ? i : i - 2];
    const bool in_place = s.src == s.dst && s.src_token == s.dst_token && s.src_head == s.dst_head;
    Job& j = a.job[i];
    j.src = s.src;
    j.dst = s.dst;
    j.src_token = (uint32_t)s.src_token;
    j.src_head = (uint32_t)s.src_head;
    j.dst_token = (uint32_t)s.dst_token;
    j.dst_head = (uint32_t)s.dst_head;
    if (turns(i)) j.pieces = r->adjacent && vec ? r->rotary_dim / step : r->rotary_dim / 2 / step;
    else if (i == 4) j.pieces = head_size / step;
    else j.pieces = in_place ? 0 : (head_size - r->rotary_dim) / step;
    j.first = turns(i) || i == 4 ? 0 : r->rotary_dim;
    j.a_token = s.heads * j.pieces;
    j.by_token = make_fast_div((uint32_t)(j.a_token > 0 ? j.a_token : 1));
    j.by_head = make_fast_div((uint32_t)(j.pieces > 0 ? j.pieces : 1));
    work += j.a_token;
    read += (int64_t)j.a_token * step * size * (turns(i) && !(r->adjacent && vec) ? 2 : 1);
  }
  if (work == 0) return kOk;
  a.table = r->table;
  a.positions = positions;
  a.axis_stride = axis_stride;
  a.table_rows = r->positions;
  a.tokens = tokens;
  for (int i = 0; i < 4; ++i) a.pair_axis[i] = r->pair_axis[i];
  a.axes = r->axes;
  a.half = r->rotary_dim / 2;
  a.sign = inverse ? -1.f : 1.f;
  a.by_half = make_fast_div((uint32_t)a.half);
  // Tokens of a workgroup: a power of two, up to ten pieces a thread (30843 tokens of
  // 40 heads of 128: up to 5 112 us, 10 114, 20 123; a write of 65536 of 8 heads of 256:
  // 124, 106, 115), fewer where that leaves less than 512 workgroups (a write of 32 MB:
  // 14.1 us, with 1024 16.3; 24 MB of 8 heads of 256: 11.7, 14.1; of 40 heads of 128:
  // 12.0, 10.7).
  int block = kMaxTokens;
  while (block > 1 && (block * work > 10 * kRotThreads || (tokens + block - 1) / block < 512)) block /= 2;
  a.block_tokens = block;
  if ((tokens + block - 1) / block > INT32_MAX) return kErrInvalidArgument;
  // More than the last-level cache holds, read and written: rows go past the caches
  // (7 heads of 256, 64 MB read: 32 us past them, 25 through; 128 MB 56.5 both; 192
  // MB 81.5, 86.5; 1 GB 411, 428).
  const bool once = 2 * tokens * read > kLastCache;
  if (dtype == OSCAR_BF16) launch_typed<__bf16>(a, vec, once, r->adjacent != 0, stream);
  else if (dtype == OSCAR_FP16) launch_typed<_Float16>(a, vec, once, r->adjacent != 0, stream);
  else launch_typed<float>(a, vec, once, r->adjacent != 0, stream);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace
}  // namespace oscar

extern "C" int oscar_rotate_positions(const oscar_rotary* rotary, const int64_t* positions,
                                      int64_t position_axis_stride, int64_t num_tokens, const oscar_heads* query,
                                      const oscar_heads* query_out, const oscar_heads* key,
                                      const oscar_heads* key_out, int32_t head_size, int32_t dtype, int32_t inverse,
                                      oscar_stream_t stream) {
  if ((query != nullptr && query->num_heads != 0 && query_out == nullptr) ||
      (key != nullptr && key->num_heads != 0 && key_out == nullptr))
    return oscar::kErrInvalidArgument;
  return oscar::run(rotary, positions, position_axis_stride, num_tokens, query, query_out, key, key_out, nullptr,
                    nullptr, nullptr, head_size, dtype, inverse, stream);
}

extern "C" int oscar_append_rotated(const oscar_rotary* rotary, const int64_t* positions,
                                    int64_t position_axis_stride, int64_t num_tokens, const oscar_heads* query,
                                    const oscar_heads* query_out, const oscar_heads* key, const oscar_heads* value,
                                    const oscar_plain_cache* cache, const int64_t* slot_mapping,
                                    oscar_stream_t stream) {
  const int status = oscar::check_plain_cache(cache);
  if (status != oscar::kOk) return status;
  if (key == nullptr || value == nullptr || key->num_heads != cache->num_kv_heads ||
      value->num_heads != cache->num_kv_heads || (num_tokens > 0 && slot_mapping == nullptr) ||
      (query != nullptr && query->num_heads != 0 && query_out == nullptr))
    return oscar::kErrInvalidArgument;
  return oscar::run(rotary, positions, position_axis_stride, num_tokens, query, query_out, key, nullptr, value, cache,
                    slot_mapping, cache->head_size, cache->dtype, 0, stream);
}
