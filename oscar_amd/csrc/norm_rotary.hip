// Norms of query and key heads with their position rotation, in one pass: to rows
// of their own (oscar_norm_rotate), with the gradient (oscar_norm_rotate_backward),
// and on the way to a paged cache, plain (oscar_append_normed) or of 8 bits
// (oscar_append_quantized, with or without norms).
//
// A head x of D features becomes
//   y = R(p) [ r x (w + offset) ],   r = 1 / sqrt(sum x^2 / D + eps),
// R the rotation of its first rotary_dim features by its token's positions.  With
// h = R(p)^T g, u = h (w + offset) and x^ = r x, the gradient is
//   dx = r (u - x^ sum(u x^) / D),   dw = sum over heads and tokens of h x^.
// All of it is fp32 arithmetic, one rounding to the rows' type at the end.
//
// (The sum is of fp32 squares: of a head whose values pass 1e18 it is an infinity, and the
// head becomes zeros.)
//
// Every value is read once and written once, so memory bounds the kernels, and for a
// few tokens their latency.  A group of lanes takes a head (16 features a lane in two
// pieces of 8, pairs that turn together in one lane), so its sums are a few
// exchanges inside 16 lanes; the tokens' cosines and the kind's weights go through LDS
// (as loads of each lane's own, sixteen for four rows, 9256 tokens take 20.0 us for
// 17.4, 30843 with the gradient 395 for 356).
// Measured: one token of 6 + 1 heads of 256 3.8 us; 9256 tokens (66 MB, in the last-level
// cache) 15.7, 4.2 TB/s; 30843 of 32 + 8 heads of 128 110 (632 MB, 5.7 TB/s), their
// gradient 181 (947 MB, 5.2 TB/s) and the weights' sums 6.9; the write of 65536 tokens of
// 6 + 1 + 1 heads of 256 to 8 bits 115 (503 MB, 4.4 TB/s), to plain pages 125 (537 MB, 4.3
// TB/s; turned alone 103).
#include "plain_cache.h"
#include "quant_cache.h"
#include "row_span.h"

#include <algorithm>
#include <type_traits>

namespace oscar {
namespace {

constexpr int kNormThreads = 256;
constexpr int kMaxTokens = 64;             // of a workgroup at a time,
constexpr int kMaxTurns = 4096;            // and their cosines and sines
constexpr int kMaxRotary = 256;
constexpr int64_t kLastCache = 256ll << 20;      // bytes
// Workgroups of the gradient, at most (1024: 30843 tokens' step 357 us for 297).
constexpr int kBackBlocks = 4096;

enum Target { kRows, kPlain, kQuant };

// What a launch does with one kind of rows: workgroups of its own, block_tokens tokens each.
struct NormJob {
  const uint8_t* src;
  uint8_t* dst;            // rows of their own, or a cache
  const uint8_t* grad;     // of the gradient: the outputs'
  const void* weight;      // null: no norm
  uint32_t src_token, src_head, dst_token, dst_head, grad_token, grad_head;   // bytes; in a cache dst_token is not used
  int32_t heads, half;     // half: rotary_dim / 2, or 0 for rows that do not turn
  int32_t block_tokens, first_block;
  FastDiv by_heads;
};
enum { kQuery, kKey, kValue, kJobs };

struct NormArgs {
  NormJob job[kJobs];
  const float* table;
  const int64_t* positions;
  int64_t axis_stride, table_rows, tokens;
  uint64_t pair_axis[4];
  const int64_t* slots;
  int64_t num_slots, k_page, k_token, v_page, v_token;
  uint8_t* exponents;      // [page][head][token][K | V]
  int32_t block_size, block_shift;         // shift: log2, or -1
  int32_t low, high;       // exponents
  int32_t axes, half;      // half: rotary_dim / 2
  int32_t adjacent;
  int32_t d, lanes, lane_shift;            // lanes of a head
  int32_t weight_type;
  float eps, offset, per_d;
  float* partials;         // of the weights' gradients: [workgroup][D], queries' first
  FastDiv by_half;
};

// Sum and maximum over a group of `lanes` (a power of two up to 16, or 64), in all of them.
template <int kCtrl>
__device__ __forceinline__ float lane_of(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xF, 0xF, true));
}
template <typename F>
__device__ __forceinline__ float over_group(float x, int lanes, F&& f) {
  if (lanes > 1) x = f(x, lane_of<0xB1>(x));           // lane ^ 1
  if (lanes > 2) x = f(x, lane_of<0x4E>(x));           // lane ^ 2
  if (lanes > 4) x = f(x, lane_of<0x141>(x));          // 7 - lane of 8
  if (lanes > 8) x = f(x, lane_of<0x140>(x));          // 15 - lane of 16
  if (lanes > 16) {
    x = f(x, __shfl_xor(x, 16, 64));
    x = f(x, __shfl_xor(x, 32, 64));
  }
  return x;
}
__device__ __forceinline__ float group_sum(float x, int lanes) {
  return over_group(x, lanes, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float group_max(float x, int lanes) {
  return over_group(x, lanes, [](float a, float b) { return fmaxf(a, b); });
}

// A lane's part of a head: kSlots places, each two pieces of kVec features in the order
// of memory.  kVec is 8 where rows, strides and pairs are multiples of 16 bytes, else 1
// (a model's head size and projection decide: 65536 tokens of 6 + 1 heads of 256 111 us in
// pieces, 177 off 16 bytes or with rotary_dim 56, 2.65 TB/s; one token 3.9, 4.4).  Pairs
// that turn together are both of one lane: the pieces' features of one index, or, where pairs
// are adjacent and kVec is 8, neighbours in a piece.
template <int kVec>
struct Part {
  static constexpr int kSlots = kVec == 8 ? 1 : 2, kPairs = kSlots * kVec;
  float x[2][kPairs];
};

// Where place u of a head lies: its first features, and whether it turns.
struct Place {
  int first, second;
  bool there, turns;
};
template <int kVec>
__device__ __forceinline__ Place place_of(const NormArgs& a, int half, int u) {
  Place p;
  p.there = 2 * kVec * u < a.d;
  p.turns = kVec * u < half;
  const bool halves = p.turns && a.adjacent == 0;
  p.first = halves ? kVec * u : 2 * kVec * u;
  p.second = halves ? half + kVec * u : 2 * kVec * u + kVec;
  return p;
}

template <typename T, int kVec, bool kOnce>
struct Piece8 {
  typedef T Row __attribute__((ext_vector_type(8)));
  u32x4 c[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* at) {
    const u32x4* p = reinterpret_cast<const u32x4*>(at);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) c[i] = kOnce ? __builtin_nontemporal_load(p + i) : p[i];
  }
  __device__ __forceinline__ void get(float* x) const {
    Row r;
    __builtin_memcpy(&r, &c, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)r[i];
  }
  __device__ __forceinline__ void put(const float* x) {
    Row r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)x[i];
    __builtin_memcpy(&c, &r, sizeof(c));
  }
  __device__ __forceinline__ void store(T* at) const {
    u32x4* p = reinterpret_cast<u32x4*>(at);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      if constexpr (kOnce) __builtin_nontemporal_store(c[i], p + i);
      else p[i] = c[i];
    }
  }
};
template <typename T, bool kOnce>
struct Piece8<T, 1, kOnce> {
  T c;
  __device__ __forceinline__ void load(const T* at) { c = *at; }
  __device__ __forceinline__ void get(float* x) const { *x = (float)c; }
  __device__ __forceinline__ void put(const float* x) { c = (T)*x; }
  __device__ __forceinline__ void store(T* at) const { *at = c; }
};

// A lane's part as it stands in memory.
template <typename T, int kVec, bool kOnce>
struct RawPart {
  Piece8<T, kVec, kOnce> p[Part<kVec>::kSlots][2];
  __device__ __forceinline__ void load(const T* row, const Place (&at)[Part<kVec>::kSlots]) {
#pragma unroll
    for (int s = 0; s < Part<kVec>::kSlots; ++s)
      if (at[s].there) {
        p[s][0].load(row + at[s].first);
        p[s][1].load(row + at[s].second);
      }
  }
  // Its values (zeros where the lane has none).
  __device__ __forceinline__ void get(const Place (&at)[Part<kVec>::kSlots], Part<kVec>& f) const {
#pragma unroll
    for (int s = 0; s < Part<kVec>::kSlots; ++s) {
      if (at[s].there) {
        p[s][0].get(&f.x[0][kVec * s]);
        p[s][1].get(&f.x[1][kVec * s]);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) f.x[0][kVec * s + i] = f.x[1][kVec * s + i] = 0.f;
      }
    }
  }
};
template <typename T, int kVec, bool kOnce>
__device__ __forceinline__ void store_part(T* row, const Place (&at)[Part<kVec>::kSlots], const Part<kVec>& f) {
#pragma unroll
  for (int s = 0; s < Part<kVec>::kSlots; ++s)
    if (at[s].there) {
      Piece8<T, kVec, kOnce> p, q;
      p.put(&f.x[0][kVec * s]);
      q.put(&f.x[1][kVec * s]);
      p.store(row + at[s].first);
      q.store(row + at[s].second);
    }
}

// Eight (or one) consecutive floats of LDS.
template <int kVec>
__device__ __forceinline__ void read_floats(const float* from, float* to) {
  if constexpr (kVec == 8) {
    const floatx4 lo = *reinterpret_cast<const floatx4*>(from), hi = *reinterpret_cast<const floatx4*>(from + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = lo[i], to[4 + i] = hi[i];
  } else {
    *to = *from;
  }
}

// R(p) x of a part, with the cosines and sines [cos | sin] of its token at `cs`; kBack:
// R(p)^T x.
template <int kVec, bool kAdjacent, bool kBack>
__device__ __forceinline__ void turn_part(const float* cs, int half, const Place (&at)[Part<kVec>::kSlots], int u0,
                                          int lanes, Part<kVec>& f) {
#pragma unroll
  for (int s = 0; s < Part<kVec>::kSlots; ++s)
    if (at[s].turns) {
      float c[kVec], sn[kVec];
      read_floats<kVec>(cs + kVec * (u0 + s * lanes), c);
      read_floats<kVec>(cs + half + kVec * (u0 + s * lanes), sn);
      auto turn = [&](float& x1, float& x2, int i) __attribute__((always_inline)) {
        const float a = x1, b = x2, t = kBack ? -sn[i] : sn[i];
        x1 = a * c[i] - b * t;
        x2 = b * c[i] + a * t;
      };
      if constexpr (kVec == 8 && kAdjacent) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          turn(f.x[0][2 * i], f.x[0][2 * i + 1], i);
          turn(f.x[1][2 * i], f.x[1][2 * i + 1], 4 + i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) turn(f.x[0][kVec * s + i], f.x[1][kVec * s + i], i);
      }
    }
}

struct TokenState {
  float cs[kMaxTurns];                     // [token][cos | sin]
  float weight[256];                       // weight + offset
  int64_t at[kMaxTokens], at_e[kMaxTokens];        // byte offsets of the slot and of its power
  int live[kMaxTokens];
};

// weight + offset of a kind (1 where there is no norm).
__device__ __forceinline__ void collect_weights(const NormArgs& a, const void* weight, TokenState& st) {
  const int f = (int)threadIdx.x;
  if (f >= a.d) return;
  float v = 1.f;
  if (weight != nullptr) {
    if (a.weight_type == OSCAR_FP32) v = static_cast<const float*>(weight)[f];
    else if (a.weight_type == OSCAR_BF16) v = (float)static_cast<const __bf16*>(weight)[f];
    else v = (float)static_cast<const _Float16*>(weight)[f];
    v += a.offset;
  }
  st.weight[f] = v;
}
template <int kVec>
__device__ __forceinline__ void load_weights(const float* from, const Place (&at)[Part<kVec>::kSlots], Part<kVec>& w) {
#pragma unroll
  for (int s = 0; s < Part<kVec>::kSlots; ++s) {
    if (at[s].there) {
      read_floats<kVec>(from + at[s].first, &w.x[0][kVec * s]);
      read_floats<kVec>(from + at[s].second, &w.x[1][kVec * s]);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) w.x[0][kVec * s + i] = w.x[1][kVec * s + i] = 0.f;
    }
  }
}

// The tokens' cosines and sines (of rows that turn), whether their positions exist, and,
// in a cache, their slots.
__device__ __forceinline__ void collect_tokens(const NormArgs& a, const NormJob& j, bool cached, bool value,
                                               int64_t tok0, int tokens, TokenState& st) {
  const int tid = (int)threadIdx.x, width = 2 * a.half;
  for (int i = tid; i < tokens * j.half; i += kNormThreads) {
    const int t = (int)fast_div((uint32_t)i, a.by_half);
    const int p = i - t * a.half;
    const int axis = (int)(a.pair_axis[p >> 5] >> (2 * (p & 31))) & 3;
    const int64_t pos = a.positions[axis * a.axis_stride + tok0 + t];
    const float* row = a.table + (pos >= 0 && pos < a.table_rows ? pos : 0) * width;
    st.cs[t * width + p] = row[p];
    st.cs[t * width + a.half + p] = row[a.half + p];
  }
  if (tid < tokens) {
    bool in = true;
    for (int x = 0; x < a.axes; ++x) {
      const int64_t pos = a.positions[x * a.axis_stride + tok0 + tid];
      in = in && pos >= 0 && pos < a.table_rows;
    }
    if (cached) {
      const int64_t slot = a.slots[tok0 + tid];
      const bool write = slot >= 0 && slot < a.num_slots;
      const int64_t s = write ? slot : 0;
      const int64_t page = a.block_shift >= 0 ? s >> a.block_shift : s / a.block_size;
      const int64_t in_page = s - page * a.block_size;
      st.at[tid] = value ? page * a.v_page + in_page * a.v_token : page * a.k_page + in_page * a.k_token;
      st.at_e[tid] = 2 * (page * j.heads * a.block_size + in_page) + (value ? 1 : 0);
      in = in && write;
    }
    st.live[tid] = in;
  }
}

// 1 / sqrt(x); the instruction takes no subnormal numbers.
__device__ __forceinline__ float inverse_root(float x) {
  const bool tiny = x < 1.2e-29f;          // 2^-96
  return __builtin_amdgcn_rsqf(tiny ? x * 0x1p64f : x) * (tiny ? 0x1p32f : 1.f);
}

// One row of 8 bits: the power of two, its byte, and the codes.
template <int kVec>
__device__ __forceinline__ void store_codes(const NormArgs& a, const Part<kVec>& f,
                                            const Place (&at)[Part<kVec>::kSlots], bool first_lane, uint8_t* row,
                                            uint8_t* exponent) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < Part<kVec>::kPairs; ++i) {
    top = fmaxf(top, finite_size(f.x[0][i]));
    top = fmaxf(top, finite_size(f.x[1][i]));
  }
  const int e = row_exponent(group_max(top, a.lanes), a.low, a.high);
  const float scale = power_of_two(-e), most = e == a.high ? 240.f : 448.f;
  if (first_lane) *exponent = (uint8_t)(e + 127);
#pragma unroll
  for (int s = 0; s < Part<kVec>::kSlots; ++s) {
    if (!at[s].there) continue;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint8_t* to = row + (p == 0 ? at[s].first : at[s].second);
      if constexpr (kVec == 8) {
        *reinterpret_cast<u32x2*>(to) = u32x2{codes4(&f.x[p][0], scale, most), codes4(&f.x[p][4], scale, most)};
      } else {
        *to = (uint8_t)code1(f.x[p][s], scale, most);
      }
    }
  }
}

// A row of a workgroup's job: `lanes` lanes each, the next one's loads on their way while
// one is computed.
template <typename T, int kVec, bool kOnce>
struct RowWork {
  RawPart<T, kVec, kOnce> x;
  int token, head;
};
template <typename T, int kVec, bool kOnce>
__device__ __forceinline__ void fetch_row(const NormJob& j, int64_t tok0, int idx,
                                          const Place (&at)[Part<kVec>::kSlots], RowWork<T, kVec, kOnce>& w) {
  w.token = (int)fast_div((uint32_t)idx, j.by_heads);
  w.head = idx - w.token * j.heads;
  w.x.load(reinterpret_cast<const T*>(j.src + tok0 * j.src_token + (uint64_t)(uint32_t)w.token * j.src_token +
                                      (uint64_t)(uint32_t)w.head * j.src_head), at);
}

template <typename T, int kVec, bool kAdjacent, int kTarget, bool kOnce>
__global__ __launch_bounds__(kNormThreads) void norm_kernel(NormArgs a) {
  constexpr int kSlots = Part<kVec>::kSlots, kPairs = Part<kVec>::kPairs;
  __shared__ __attribute__((aligned(16))) TokenState st;
  const int block = (int)blockIdx.x;
  const int kind = block >= a.job[kValue].first_block ? kValue : block >= a.job[kKey].first_block ? kKey : kQuery;
  const NormJob& j = a.job[kind];
  const int tid = (int)threadIdx.x;
  const int group = tid >> a.lane_shift, u0 = tid & (a.lanes - 1), groups = kNormThreads >> a.lane_shift;
  const int64_t tok0 = (int64_t)(block - j.first_block) * j.block_tokens;
  const int tokens = (int)min((int64_t)j.block_tokens, a.tokens - tok0), count = tokens * j.heads;
  const bool cached = kTarget != kRows && kind != kQuery;
  Place at[kSlots];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) at[s] = place_of<kVec>(a, j.half, u0 + s * a.lanes);

  typedef RowWork<T, kVec, kOnce> Work;
  auto finish = [&](const Work& w, const Part<kVec>& weight) {
    if (st.live[w.token] == 0) return;
    Part<kVec> f;
    w.x.get(at, f);
    if (j.weight != nullptr) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) sum += f.x[0][i] * f.x[0][i] + f.x[1][i] * f.x[1][i];
      const float r = inverse_root(group_sum(sum, a.lanes) * a.per_d + a.eps);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        f.x[0][i] = f.x[0][i] * r * weight.x[0][i];
        f.x[1][i] = f.x[1][i] * r * weight.x[1][i];
      }
    }
    turn_part<kVec, kAdjacent, false>(st.cs + w.token * 2 * a.half, a.half, at, u0, a.lanes, f);
    uint8_t* dst = j.dst + (uint64_t)(uint32_t)w.head * j.dst_head;
    dst += cached ? st.at[w.token] : tok0 * j.dst_token + (uint64_t)(uint32_t)w.token * j.dst_token;
    if (kTarget == kQuant && cached)
      store_codes<kVec>(a, f, at, u0 == 0, dst, a.exponents + st.at_e[w.token] + 2 * (int64_t)w.head * a.block_size);
    else
      store_part<T, kVec, kOnce>(reinterpret_cast<T*>(dst), at, f);
  };
  Work now;
  if (group < count) fetch_row(j, tok0, group, at, now);
  collect_weights(a, j.weight, st);
  collect_tokens(a, j, cached, kind == kValue, tok0, tokens, st);
  __syncthreads();
  Part<kVec> weight;
  load_weights<kVec>(st.weight, at, weight);
  for (int idx = group; idx < count; idx += groups) {
    Work next;
    if (idx + groups < count) fetch_row(j, tok0, idx + groups, at, next);
    finish(now, weight);
    now = next;
  }
}

// The gradient.  A workgroup goes from block to block of a kind's tokens, a lane's sums for
// its weights in registers; at the end they meet in LDS and leave one partial a
// workgroup, which weight_kernel adds up in order.
template <typename T, int kVec, bool kAdjacent, bool kOnce>
__global__ __launch_bounds__(kNormThreads) void backward_kernel(NormArgs a) {
  constexpr int kSlots = Part<kVec>::kSlots, kPairs = Part<kVec>::kPairs;
  constexpr size_t kSums = kNormThreads * 2 * kPairs * 4;      // [group][D]
  __shared__ __attribute__((aligned(16))) uint8_t smem[kSums > sizeof(TokenState) ? kSums : sizeof(TokenState)];
  TokenState& st = *reinterpret_cast<TokenState*>(smem);
  float* const all = reinterpret_cast<float*>(smem);
  const int kind = (int)blockIdx.x >= a.job[kKey].first_block ? kKey : kQuery;
  const NormJob& j = a.job[kind];
  const int stride = (kind == kKey ? (int)gridDim.x : a.job[kKey].first_block) - j.first_block;
  const int tid = (int)threadIdx.x;
  const int group = tid >> a.lane_shift, u0 = tid & (a.lanes - 1), groups = kNormThreads >> a.lane_shift;
  Place at[kSlots];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) at[s] = place_of<kVec>(a, j.half, u0 + s * a.lanes);
  struct Work {
    RowWork<T, kVec, kOnce> row;
    RawPart<T, kVec, kOnce> g;
  };
  Part<kVec> sums, weight;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) sums.x[0][i] = sums.x[1][i] = 0.f;
  collect_weights(a, j.weight, st);
  __syncthreads();
  load_weights<kVec>(st.weight, at, weight);
  for (int64_t block = (int)blockIdx.x - j.first_block; block * j.block_tokens < a.tokens; block += stride) {
    const int64_t tok0 = block * j.block_tokens;
    const int tokens = (int)min((int64_t)j.block_tokens, a.tokens - tok0), count = tokens * j.heads;
    auto fetch = [&](int idx, Work& w) {
      fetch_row(j, tok0, idx, at, w.row);
      w.g.load(reinterpret_cast<const T*>(j.grad + tok0 * j.grad_token + (uint64_t)(uint32_t)w.row.token * j.grad_token +
                                          (uint64_t)(uint32_t)w.row.head * j.grad_head), at);
    };
    auto finish = [&](const Work& w) {
      Part<kVec> x, u;
      w.row.x.get(at, x);
      w.g.get(at, u);
      const bool live = st.live[w.row.token] != 0;
      turn_part<kVec, kAdjacent, true>(st.cs + w.row.token * 2 * a.half, a.half, at, u0, a.lanes, u);
      float xx = 0.f, ux = 0.f;
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          xx += x.x[e][i] * x.x[e][i];
          ux += x.x[e][i] * u.x[e][i] * weight.x[e][i];
        }
      const float r = inverse_root(group_sum(xx, a.lanes) * a.per_d + a.eps);
      const float inner = group_sum(ux, a.lanes) * a.per_d * r;
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float unit = x.x[e][i] * r, h = u.x[e][i];
          sums.x[e][i] += live ? h * unit : 0.f;
          u.x[e][i] = live ? r * (h * weight.x[e][i] - unit * inner) : 0.f;
        }
      if (j.dst != nullptr)
        store_part<T, kVec, kOnce>(
            reinterpret_cast<T*>(j.dst + tok0 * j.dst_token + (uint64_t)(uint32_t)w.row.token * j.dst_token +
                                 (uint64_t)(uint32_t)w.row.head * j.dst_head), at, u);
    };
    Work now;
    if (group < count) fetch(group, now);
    __syncthreads();                        // (the block before this one is done with the cosines)
    collect_tokens(a, j, false, false, tok0, tokens, st);
    __syncthreads();
    for (int idx = group; idx < count; idx += groups) {
      Work next;
      if (idx + groups < count) fetch(idx + groups, next);
      finish(now);
      now = next;
    }
  }
  if (a.partials == nullptr) return;
  // The groups' sums: a thread to a feature.
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kSlots; ++s)
    if (at[s].there)
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        all[group * a.d + at[s].first + i] = sums.x[0][kVec * s + i];
        all[group * a.d + at[s].second + i] = sums.x[1][kVec * s + i];
      }
  __syncthreads();
  if (tid < a.d) {
    float sum = 0.f;
    for (int g = 0; g < groups; ++g) sum += all[g * a.d + tid];
    a.partials[(int64_t)blockIdx.x * a.d + tid] = sum;
  }
}

// The weights' gradients: the workgroups' partials of 16 features, 64 threads to each,
// eight loads at once.
constexpr int kWeightParts = 64;
__global__ __launch_bounds__(16 * kWeightParts) void weight_kernel(const float* partials, int queries, int keys, int d,
                                                                   void* query, void* key, int weight_type) {
  __shared__ float red[kWeightParts][17];
  const int f = 16 * (int)blockIdx.x + ((int)threadIdx.x & 15), part = (int)threadIdx.x >> 4, k = (int)blockIdx.y;
  void* const out = k == 0 ? query : key;
  if (out == nullptr) return;
  const int blocks = k == 0 ? queries : keys;
  const float* const from = partials + (k == 0 ? 0 : (int64_t)queries * d);
  float sum[8] = {};
  if (f < d)
    for (int b = part; b < blocks; b += 8 * kWeightParts)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = b + i * kWeightParts;
        const float x = from[(int64_t)min(at, blocks - 1) * d + f];
        sum[i] += at < blocks ? x : 0.f;
      }
  red[part][threadIdx.x & 15] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
  __syncthreads();
  if (part != 0 || f >= d) return;
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < kWeightParts; ++i) total += red[i][threadIdx.x];
  if (weight_type == OSCAR_FP32) static_cast<float*>(out)[f] = total;
  else if (weight_type == OSCAR_BF16) static_cast<__bf16*>(out)[f] = (__bf16)total;
  else static_cast<_Float16*>(out)[f] = (_Float16)total;
}

// ---------------------------------------------------------------- host
int dtype_size(int32_t dtype) { return dtype == OSCAR_FP32 ? 4 : 2; }

struct Rows {
  uint8_t* at;
  int64_t token, head;     // bytes
  int32_t heads;
};

RowSpan span_of(const Rows& s, int64_t tokens, int64_t row) {
  return RowSpan{(uint64_t)(uintptr_t)s.at, s.token, s.head, tokens, s.heads, row};
}

// (Strides between rows of which there is one mean nothing.)
int make_rows(Rows& s, const oscar_heads* x, int64_t tokens, int size, bool& vec) {
  if (x == nullptr || x->num_heads == 0) return kOk;
  if (x->data == nullptr || x->num_heads < 0 || x->num_heads > (1 << 16)) return kErrInvalidArgument;
  s.at = static_cast<uint8_t*>(x->data);
  s.token = tokens > 1 ? x->token_stride : 0;
  s.head = x->num_heads > 1 ? x->head_stride : 0;
  s.heads = x->num_heads;
  for (int64_t* const y : {&s.token, &s.head}) {
    if (*y < 0 || *y > UINT32_MAX / size) return kErrUnsupportedGeometry;
    *y *= size;
  }
  vec = vec && ((uintptr_t)s.at | (uintptr_t)s.token | (uintptr_t)s.head) % 16 == 0;
  return kOk;
}

int check_norm(const oscar_rotary* r, const oscar_head_norm* n, int64_t tokens, int32_t head_size, int32_t dtype) {
  if (tokens < 0 || r == nullptr || r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > kMaxRotary ||
      r->axes < 1 || r->axes > 4 || r->positions < 1 || dtype < OSCAR_BF16 || dtype > OSCAR_FP32 || n == nullptr ||
      n->weight_dtype < OSCAR_BF16 || n->weight_dtype > OSCAR_FP32 || !(n->eps >= 0.f) || !(n->eps < 3.0e38f) ||
      !(n->offset > -3.0e38f) || !(n->offset < 3.0e38f))
    return kErrInvalidArgument;
  if (head_size < r->rotary_dim || head_size % 2 || head_size > 256) return kErrUnsupportedHeadDim;
  for (int j = 0; j < r->rotary_dim / 2; ++j)
    if ((int)((r->pair_axis[j >> 5] >> (2 * (j & 31))) & 3) >= r->axes) return kErrInvalidArgument;
  return kOk;
}

// What all launches have in common; `vec`: rows in pieces of 16 bytes.
void fill_args(NormArgs& a, const oscar_rotary* r, const oscar_head_norm* n, const int64_t* positions,
               int64_t axis_stride, int64_t tokens, int32_t head_size, bool vec) {
  a.table = r->table;
  a.positions = positions;
  a.axis_stride = axis_stride;
  a.table_rows = r->positions;
  a.tokens = tokens;
  for (int i = 0; i < 4; ++i) a.pair_axis[i] = r->pair_axis[i];
  a.axes = r->axes;
  a.half = r->rotary_dim / 2;
  a.adjacent = r->adjacent != 0;
  a.d = head_size;
  a.lanes = 64;
  if (vec)
    for (a.lanes = 1; a.lanes < head_size / 16;) a.lanes *= 2;
  for (a.lane_shift = 0; 1 << a.lane_shift < a.lanes;) ++a.lane_shift;
  a.weight_type = n->weight_dtype;
  a.eps = n->eps;
  a.offset = n->offset;
  a.per_d = 1.f / (float)head_size;
  a.by_half = make_fast_div((uint32_t)a.half);
  a.job[kQuery].weight = n->query_weight;
  a.job[kKey].weight = n->key_weight;
  for (int i = 0; i < kJobs; ++i) {
    a.job[i].by_heads = make_fast_div((uint32_t)(a.job[i].heads > 0 ? a.job[i].heads : 1));
    a.job[i].half = i == kValue ? 0 : a.half;
  }
}

bool pieces_of_16(const oscar_rotary* r, int32_t head_size) { return head_size % 16 == 0 && r->rotary_dim % 16 == 0; }

// Tokens of a workgroup of a kind: a power of two, up to kRounds heads a group of lanes (8:
// 30843 tokens' gradient step 357 us for 303), fewer where that leaves less than 256
// workgroups (512: 2000 tokens of 7 heads 7.7 us for 6.4), more than 8 only where there are
// 2048 of them (where less do: 9256 tokens 17.5 us for 16.1).
constexpr int kRounds = 4;
int tokens_a_block(int64_t tokens, const NormJob& j, int lanes) {
  int block = kMaxTokens;
  while (block > 1 && (block * (int64_t)j.heads * lanes > kRounds * kNormThreads || 2 * j.half * block > kMaxTurns ||
                       (tokens + block - 1) / block < (block > 8 ? 2048 : 256)))
    block /= 2;
  return block;
}
int64_t blocks_of(const NormJob& j, int64_t tokens) {
  return j.heads == 0 ? 0 : (tokens + j.block_tokens - 1) / j.block_tokens;
}

template <typename T, int kTarget>
void launch_norm(const NormArgs& a, uint32_t blocks, bool vec, bool once, hipStream_t stream) {
  // (single values of adjacent pairs and of halves differ in their places alone)
  const auto kernel = !vec                 ? &norm_kernel<T, 1, false, kTarget, false>
                      : a.adjacent && once ? &norm_kernel<T, 8, true, kTarget, true>
                      : a.adjacent         ? &norm_kernel<T, 8, true, kTarget, false>
                      : once               ? &norm_kernel<T, 8, false, kTarget, true>
                                           : &norm_kernel<T, 8, false, kTarget, false>;
  kernel<<<blocks, kNormThreads, 0, stream>>>(a);
}

// kTarget's cache: plain or quant.
template <int kTarget>
int run_norm(const oscar_rotary* r, const oscar_head_norm* n, const int64_t* positions, int64_t axis_stride,
             int64_t tokens, const oscar_heads* query, const oscar_heads* query_out, const oscar_heads* key,
             const oscar_heads* key_out, const oscar_heads* value, const oscar_plain_cache* plain,
             const oscar_quant_cache* quant, const int64_t* slots, int32_t head_size, int32_t dtype,
             hipStream_t stream) {
  int status = check_norm(r, n, tokens, head_size, dtype);
  if (status != kOk) return status;
  if (tokens == 0) return kOk;
  if (r->table == nullptr || positions == nullptr) return kErrInvalidArgument;
  const int size = dtype_size(dtype);
  bool vec = pieces_of_16(r, head_size);
  const oscar_heads* const in[kJobs] = {query, key, value};
  const oscar_heads* const out[kJobs] = {query_out, key_out, nullptr};
  Rows from[kJobs] = {}, to[kJobs] = {};
  for (int i = 0; i < kJobs; ++i) {
    status = make_rows(from[i], in[i], tokens, size, vec);
    if (status != kOk) return status;
    if (out[i] == nullptr || from[i].heads == 0) continue;
    status = make_rows(to[i], out[i], tokens, size, vec);
    if (status != kOk) return status;
    if (to[i].heads != from[i].heads) return kErrInvalidArgument;
  }
  // An output that is its input is read and written row by row by the same lanes; of any
  // other rows that it shares memory with, some would be read after they are written.
  const int64_t row = (int64_t)head_size * size;
  for (int i = 0; i < 2; ++i) {
    if (to[i].heads == 0) continue;
    const RowSpan x = span_of(to[i], tokens, row);
    for (int j = 0; j < kJobs; ++j) {
      const RowSpan y = span_of(from[j], tokens, row);
      if (!(i == j && same_rows(x, y)) && !rows_apart(x, y)) return kErrOverlap;
    }
    if (i == 0 && !rows_apart(x, span_of(to[1], tokens, row))) return kErrOverlap;
  }
  NormArgs a{};
  int64_t heads = 0;
  for (int i = 0; i < kJobs; ++i) {
    NormJob& j = a.job[i];
    j.src = from[i].at;
    j.src_token = (uint32_t)from[i].token;
    j.src_head = (uint32_t)from[i].head;
    j.dst = to[i].at;
    j.dst_token = (uint32_t)to[i].token;
    j.dst_head = (uint32_t)to[i].head;
    j.heads = from[i].heads;
    heads += j.heads;
  }
  if (heads == 0) return kOk;
  if (kTarget != kRows) {
    int64_t pages, k_head, v_head;
    if (kTarget == kPlain) {
      a.job[kKey].dst = static_cast<uint8_t*>(plain->k);
      a.job[kValue].dst = static_cast<uint8_t*>(plain->v);
      pages = plain->num_pages, a.block_size = plain->block_size;
      a.k_page = plain->k_stride_page, a.k_token = plain->k_stride_token, k_head = plain->k_stride_head;
      a.v_page = plain->v_stride_page, a.v_token = plain->v_stride_token, v_head = plain->v_stride_head;
    } else {
      a.job[kKey].dst = static_cast<uint8_t*>(quant->k);
      a.job[kValue].dst = static_cast<uint8_t*>(quant->v);
      pages = quant->num_pages, a.block_size = quant->block_size;
      a.k_page = quant->k_stride_page, a.k_token = quant->k_stride_token, k_head = quant->k_stride_head;
      a.v_page = quant->v_stride_page, a.v_token = quant->v_stride_token, v_head = quant->v_stride_head;
      a.exponents = quant->exponents;
      a.low = exponent_range(dtype).low;
      a.high = exponent_range(dtype).high;
    }
    a.job[kKey].dst_head = (uint32_t)k_head;
    a.job[kValue].dst_head = (uint32_t)v_head;
    a.slots = slots;
    a.num_slots = pages * a.block_size;
    a.block_shift = -1;
    for (int s = 0; s < 31; ++s)
      if (a.block_size == (1 << s)) a.block_shift = s;
  }
  fill_args(a, r, n, positions, axis_stride, tokens, head_size, vec);
  int64_t blocks = 0;
  for (int i = 0; i < kJobs; ++i) {
    NormJob& j = a.job[i];
    j.block_tokens = tokens_a_block(tokens, j, a.lanes);
    j.first_block = (int32_t)blocks;
    blocks += blocks_of(j, tokens);
    if (blocks > INT32_MAX) return kErrInvalidArgument;
  }
  // More than the last-level cache holds, read and written: rows go past the caches.
  const bool once = 2 * tokens * heads * row > kLastCache;
  if (dtype == OSCAR_BF16) launch_norm<__bf16, kTarget>(a, (uint32_t)blocks, vec, once, stream);
  else if (dtype == OSCAR_FP16) launch_norm<_Float16, kTarget>(a, (uint32_t)blocks, vec, once, stream);
  else if constexpr (kTarget == kRows) launch_norm<float, kTarget>(a, (uint32_t)blocks, vec, once, stream);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

template <typename T>
void launch_backward(const NormArgs& a, uint32_t blocks, bool vec, bool once, hipStream_t stream) {
  const auto kernel = !vec         ? &backward_kernel<T, 1, false, false>
                      : a.adjacent ? once ? &backward_kernel<T, 8, true, true> : &backward_kernel<T, 8, true, false>
                      : once       ? &backward_kernel<T, 8, false, true>
                                   : &backward_kernel<T, 8, false, false>;
  kernel<<<blocks, kNormThreads, 0, stream>>>(a);
}

}  // namespace
}  // namespace oscar

extern "C" int oscar_norm_rotate(const oscar_rotary* rotary, const oscar_head_norm* norm, const int64_t* positions,
                                 int64_t position_axis_stride, int64_t num_tokens, const oscar_heads* query,
                                 const oscar_heads* query_out, const oscar_heads* key, const oscar_heads* key_out,
                                 int32_t head_size, int32_t dtype, oscar_stream_t stream) {
  if ((query != nullptr && query->num_heads != 0 && query_out == nullptr) ||
      (key != nullptr && key->num_heads != 0 && key_out == nullptr))
    return oscar::kErrInvalidArgument;
  return oscar::run_norm<oscar::kRows>(rotary, norm, positions, position_axis_stride, num_tokens, query, query_out, key,
                                       key_out, nullptr, nullptr, nullptr, nullptr, head_size, dtype, stream);
}

extern "C" int oscar_append_normed(const oscar_rotary* rotary, const oscar_head_norm* norm, const int64_t* positions,
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
  return oscar::run_norm<oscar::kPlain>(rotary, norm, positions, position_axis_stride, num_tokens, query, query_out, key,
                                        nullptr, value, cache, nullptr, slot_mapping, cache->head_size, cache->dtype,
                                        stream);
}

extern "C" int oscar_append_quantized(const oscar_rotary* rotary, const oscar_head_norm* norm,
                                      const int64_t* positions, int64_t position_axis_stride, int64_t num_tokens,
                                      const oscar_heads* query, const oscar_heads* query_out, const oscar_heads* key,
                                      const oscar_heads* value, const oscar_quant_cache* cache,
                                      const int64_t* slot_mapping, oscar_stream_t stream) {
  const int status = oscar::check_quant_cache(cache);
  if (status != oscar::kOk) return status;
  if (key == nullptr || value == nullptr || key->num_heads != cache->num_kv_heads ||
      value->num_heads != cache->num_kv_heads || (num_tokens > 0 && slot_mapping == nullptr) ||
      (query != nullptr && query->num_heads != 0 && query_out == nullptr))
    return oscar::kErrInvalidArgument;
  return oscar::run_norm<oscar::kQuant>(rotary, norm, positions, position_axis_stride, num_tokens, query, query_out, key,
                                        nullptr, value, nullptr, cache, slot_mapping, cache->head_size, cache->dtype,
                                        stream);
}

extern "C" size_t oscar_norm_rotate_backward_workspace_bytes(int64_t num_tokens, int32_t head_size) {
  if (num_tokens < 1 || head_size < 2 || head_size > 256) return 0;
  return (size_t)std::min<int64_t>(num_tokens, oscar::kBackBlocks) * 2 * (size_t)head_size * 4;
}

extern "C" int oscar_norm_rotate_backward(const oscar_rotary* rotary, const oscar_head_norm* norm,
                                          const int64_t* positions, int64_t position_axis_stride, int64_t num_tokens,
                                          const oscar_heads* query, const oscar_heads* query_out_grad,
                                          const oscar_heads* query_grad, const oscar_heads* key,
                                          const oscar_heads* key_out_grad, const oscar_heads* key_grad,
                                          void* query_weight_grad, void* key_weight_grad, int32_t head_size,
                                          int32_t dtype, void* workspace, size_t workspace_size,
                                          oscar_stream_t stream) {
  using namespace oscar;
  int status = check_norm(rotary, norm, num_tokens, head_size, dtype);
  if (status != kOk) return status;
  const bool weights = query_weight_grad != nullptr || key_weight_grad != nullptr;
  const size_t need = weights ? oscar_norm_rotate_backward_workspace_bytes(num_tokens, head_size) : 0;
  if (workspace_size < need || (need > 0 && workspace == nullptr)) return kErrWorkspaceTooSmall;
  if ((uintptr_t)workspace % 4) return kErrUnsupportedGeometry;
  if (num_tokens > 0 && (rotary->table == nullptr || positions == nullptr)) return kErrInvalidArgument;
  const int size = dtype_size(dtype);
  bool vec = pieces_of_16(rotary, head_size);
  const oscar_heads* const in[2][3] = {{query, query_out_grad, query_grad}, {key, key_out_grad, key_grad}};
  const void* const weight[2] = {norm->query_weight, norm->key_weight};
  Rows rows[2][3] = {};
  int64_t heads = 0;
  for (int i = 0; i < 2; ++i) {
    for (int j = 0; j < 3; ++j) {
      status = make_rows(rows[i][j], in[i][j], num_tokens, size, vec);
      if (status != kOk) return status;
    }
    // (a kind without rows of its own has no gradient; the rows' own is left out if it is not asked for)
    if (rows[i][0].heads != rows[i][1].heads || (rows[i][2].heads != 0 && rows[i][2].heads != rows[i][0].heads) ||
        (rows[i][0].heads > 0 && weight[i] == nullptr))
      return kErrInvalidArgument;
    heads += rows[i][0].heads;
  }
  const int64_t row = (int64_t)head_size * size;
  for (int i = 0; i < 2; ++i) {
    const RowSpan x = span_of(rows[i][2], num_tokens, row);
    for (int k = 0; k < 2; ++k)
      for (int j = 0; j < 3; ++j)
        if ((i != k || j != 2) && !rows_apart(x, span_of(rows[k][j], num_tokens, row))) return kErrOverlap;
  }
  NormArgs a{};
  for (int i = 0; i < 2; ++i) {
    NormJob& j = a.job[i];
    j.src = rows[i][0].at;
    j.src_token = (uint32_t)rows[i][0].token;
    j.src_head = (uint32_t)rows[i][0].head;
    j.grad = rows[i][1].at;
    j.grad_token = (uint32_t)rows[i][1].token;
    j.grad_head = (uint32_t)rows[i][1].head;
    j.dst = rows[i][2].at;
    j.dst_token = (uint32_t)rows[i][2].token;
    j.dst_head = (uint32_t)rows[i][2].head;
    j.heads = rows[i][0].heads;
  }
  fill_args(a, rotary, norm, positions, position_axis_stride, num_tokens, head_size, vec);
  a.partials = weights ? static_cast<float*>(workspace) : nullptr;
  // Workgroups of the two kinds as their heads are, each at least one where there are rows.
  int64_t blocks[2] = {};
  for (int i = 0; i < 2; ++i) {
    NormJob& j = a.job[i];
    j.block_tokens = tokens_a_block(num_tokens, j, a.lanes);
    const int64_t share = kBackBlocks * j.heads / std::max<int64_t>(1, heads);
    blocks[i] = std::min<int64_t>(blocks_of(j, num_tokens), std::max<int64_t>(1, share));
  }
  a.job[kKey].first_block = (int32_t)blocks[0];
  if (blocks[0] + blocks[1] > 0) {
    const bool once = 3 * num_tokens * heads * row > kLastCache;
    const uint32_t grid = (uint32_t)(blocks[0] + blocks[1]);
    if (dtype == OSCAR_BF16) launch_backward<__bf16>(a, grid, vec, once, stream);
    else if (dtype == OSCAR_FP16) launch_backward<_Float16>(a, grid, vec, once, stream);
    else launch_backward<float>(a, grid, vec, once, stream);
  }
  if (weights)
    weight_kernel<<<dim3((uint32_t)(head_size + 15) / 16, 2), 16 * kWeightParts, 0, stream>>>(
        a.partials, (int)blocks[0], (int)blocks[1], head_size, query_weight_grad, key_weight_grad, norm->weight_dtype);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}
