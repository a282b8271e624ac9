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
// LDS first (each table entry read once for all heads, each pair from its own
// axis' row), while its first rows are already on their way; then every thread
// takes pieces of rows: a rotating piece is kVec pairs, a copying one kVec
// values (features past rotary_dim, and the values).
#include "plain_cache.h"

namespace oscar {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxTokens = 16;             // of a workgroup
constexpr int kMaxRotary = 256;

// Rows that a launch turns or copies: source, destination (or cache slots).
struct RowSet {
  const uint8_t* src;
  uint8_t* dst;
  int64_t src_token, src_head, dst_token, dst_head;    // bytes; in a cache dst_token is not used
  int32_t heads;
  int32_t pieces;          // of a head
  int32_t turning;         // of them, the first ones
  int32_t first;           // piece of a token at which the set starts
  FastDiv by_pieces;
};

struct RotArgs {
  RowSet set[3];           // queries, keys, values
  const float* table;
  const int64_t* positions;
  int64_t axis_stride, table_rows, tokens;
  uint64_t pair_axis[4];
  const int64_t* slots;    // null: sets have rows of their own
  int64_t num_slots, k_page, k_token, v_page, v_token;
  int32_t block_size, block_shift;         // shift: log2, or -1
  int32_t axes, half;      // rotary_dim / 2
  int32_t pieces;          // of a token
  int32_t block_tokens;
  float sign;              // of the sines
  FastDiv by_pieces, by_half;
};

template <typename T, int kVec>
struct Piece {
  typedef T Row __attribute__((ext_vector_type(kVec)));
};
template <typename T>
struct Piece<T, 1> {
  typedef T Row;
};

// One thread's piece: where it lies, and its values.
template <typename T, int kVec>
struct Work {
  typename Piece<T, kVec>::Row a, b;
  const uint8_t* src;
  int token, set, head, piece;             // set < 0: none
};

// kVec values to a load: 16 bytes where rows, strides and pairs allow, else one
// value (a model's head size and projection decide, not the caller).
template <typename T, int kVec, bool kAdjacent>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs a) {
  typedef typename Piece<T, kVec>::Row Row;
  __shared__ __attribute__((aligned(16))) float cs[kMaxTokens * kMaxRotary];   // [token][cos | sin]
  __shared__ int64_t at_k[kMaxTokens], at_v[kMaxTokens];                       // byte offset of the slot, -1: none
  __shared__ int live[kMaxTokens];
  const int tid = (int)threadIdx.x;
  const int64_t tok0 = (int64_t)blockIdx.x * a.block_tokens;
  const int tokens = (int)min((int64_t)a.block_tokens, a.tokens - tok0);
  const int count = tokens * a.pieces;
  constexpr int kPairs = kAdjacent && kVec > 1 ? kVec / 2 : kVec;     // of a turning piece
  const int width = 2 * a.half;

  auto locate = [&](int idx, Work<T, kVec>& w) {
    w.set = -1;
    if (idx >= count) return;
    w.token = (int)fast_div((uint32_t)idx, a.by_pieces);
    const int p = idx - w.token * a.pieces;
    w.set = p >= a.set[2].first ? 2 : p >= a.set[1].first ? 1 : 0;
    const RowSet& s = a.set[w.set];
    w.head = (int)fast_div((uint32_t)(p - s.first), s.by_pieces);
    w.piece = p - s.first - w.head * s.pieces;
    w.src = s.src + (tok0 + w.token) * s.src_token + (int64_t)w.head * s.src_head;
  };
  // First feature of a piece, and of its partners (features j and j + half).
  auto feature = [&](const Work<T, kVec>& w) {
    const int turning = a.set[w.set].turning;
    if (w.piece < turning) return w.piece * kVec * (kVec == 1 && kAdjacent ? 2 : 1);
    return (w.set < 2 ? width : 0) + (w.piece - turning) * kVec;
  };
  auto fetch = [&](Work<T, kVec>& w) {
    if (w.set < 0) return;
    const T* x = reinterpret_cast<const T*>(w.src) + feature(w);
    w.a = *reinterpret_cast<const Row*>(x);
    if (w.piece < a.set[w.set].turning) {
      if constexpr (!kAdjacent) w.b = *reinterpret_cast<const Row*>(x + a.half);
      else if constexpr (kVec == 1) w.b = *reinterpret_cast<const Row*>(x + 1);
    }
  };

  Work<T, kVec> next;
  locate(tid, next);
  fetch(next);

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

  for (int idx = tid; idx < count; idx += kRotThreads) {
    Work<T, kVec> w = next;
    locate(idx + kRotThreads, next);
    fetch(next);
    if (live[w.token] == 0) continue;
    const RowSet& s = a.set[w.set];
    uint8_t* dst = s.dst + (int64_t)w.head * s.dst_head;
    if (a.slots != nullptr && w.set > 0) {
      const int64_t at = w.set == 1 ? at_k[w.token] : at_v[w.token];
      if (at < 0) continue;
      dst += at;
    } else {
      dst += (tok0 + w.token) * s.dst_token;
    }
    T* y = reinterpret_cast<T*>(dst) + feature(w);
    if (w.piece < s.turning) {
      const float* c = cs + w.token * width + w.piece * kPairs;
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
        *reinterpret_cast<Row*>(y) = o;
      } else {
        Row o1, o2;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float x1 = (float)w.a[i], x2 = (float)w.b[i];
          o1[i] = (T)(x1 * c[i] - x2 * sn[i]);
          o2[i] = (T)(x2 * c[i] + x1 * sn[i]);
        }
        *reinterpret_cast<Row*>(y) = o1;
        *reinterpret_cast<Row*>(y + a.half) = o2;
      }
    } else {
      *reinterpret_cast<Row*>(y) = w.a;
    }
  }
}

template <typename T>
void launch_typed(const RotArgs& a, bool vec, bool adjacent, hipStream_t stream) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const dim3 grid((uint32_t)((a.tokens + a.block_tokens - 1) / a.block_tokens));
  if (vec && adjacent) rotary_kernel<T, kVec, true><<<grid, kRotThreads, 0, stream>>>(a);
  else if (vec) rotary_kernel<T, kVec, false><<<grid, kRotThreads, 0, stream>>>(a);
  else if (adjacent) rotary_kernel<T, 1, true><<<grid, kRotThreads, 0, stream>>>(a);
  else rotary_kernel<T, 1, false><<<grid, kRotThreads, 0, stream>>>(a);
}

int dtype_size(int32_t dtype) { return dtype == OSCAR_FP32 ? 4 : 2; }

bool fits16(const void* p, int64_t token_bytes, int64_t head_bytes) {
  return ((uintptr_t)p | (uintptr_t)token_bytes | (uintptr_t)head_bytes) % 16 == 0;
}

// Source and destination of a set; out null: cache slots.
bool make_set(RowSet& s, const oscar_heads* in, const oscar_heads* out, int size, bool& vec) {
  if (in == nullptr || in->num_heads == 0) return true;
  if (in->data == nullptr || in->num_heads < 0 || in->num_heads > (1 << 16)) return false;
  s.src = static_cast<const uint8_t*>(in->data);
  s.src_token = in->token_stride * size;
  s.src_head = in->head_stride * size;
  s.heads = in->num_heads;
  vec = vec && fits16(s.src, s.src_token, s.src_head);
  if (out != nullptr) {
    if (out->data == nullptr || out->num_heads != in->num_heads) return false;
    s.dst = static_cast<uint8_t*>(out->data);
    s.dst_token = out->token_stride * size;
    s.dst_head = out->head_stride * size;
    vec = vec && fits16(s.dst, s.dst_token, s.dst_head);
  }
  return true;
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
  if (!make_set(a.set[0], query, query_out, size, vec) || !make_set(a.set[1], key, key_out, size, vec) ||
      !make_set(a.set[2], value, nullptr, size, vec))
    return kErrInvalidArgument;
  if (cache != nullptr) {
    a.set[1].dst = static_cast<uint8_t*>(cache->k);
    a.set[1].dst_head = cache->k_stride_head;
    a.set[2].dst = static_cast<uint8_t*>(cache->v);
    a.set[2].dst_head = cache->v_stride_head;
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
  for (int i = 0; i < 3; ++i) {
    RowSet& s = a.set[i];
    const bool in_place = i < 2 && s.src == s.dst && s.src_token == s.dst_token && s.src_head == s.dst_head &&
                          !(cache != nullptr && i == 1);
    s.turning = i == 2 ? 0 : (r->adjacent ? (vec ? r->rotary_dim / step : r->rotary_dim / 2) : r->rotary_dim / 2 / step);
    s.pieces = i == 2 ? head_size / step : s.turning + (in_place ? 0 : (head_size - r->rotary_dim) / step);
    s.first = i == 0 ? 0 : a.set[i - 1].first + a.set[i - 1].heads * a.set[i - 1].pieces;
    s.by_pieces = make_fast_div((uint32_t)s.pieces);
    a.pieces += s.heads * s.pieces;
  }
  if (a.pieces == 0) return kOk;
  a.table = r->table;
  a.positions = positions;
  a.axis_stride = axis_stride;
  a.table_rows = r->positions;
  a.tokens = tokens;
  for (int i = 0; i < 4; ++i) a.pair_axis[i] = r->pair_axis[i];
  a.axes = r->axes;
  a.half = r->rotary_dim / 2;
  a.sign = inverse ? -1.f : 1.f;
  a.by_pieces = make_fast_div((uint32_t)a.pieces);
  a.by_half = make_fast_div((uint32_t)a.half);
  // Tokens of a workgroup: eight pieces a thread, one token where they are few.
  int block = (8 * kRotThreads + a.pieces - 1) / a.pieces;
  block = block > kMaxTokens ? kMaxTokens : block;
  while (block > 1 && (tokens + block - 1) / block < 1024) block /= 2;
  a.block_tokens = block;
  if ((tokens + block - 1) / block > INT32_MAX) return kErrInvalidArgument;
  if (dtype == OSCAR_BF16) launch_typed<__bf16>(a, vec, r->adjacent != 0, stream);
  else if (dtype == OSCAR_FP16) launch_typed<_Float16>(a, vec, r->adjacent != 0, stream);
  else launch_typed<float>(a, vec, r->adjacent != 0, stream);
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
