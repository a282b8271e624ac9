// Causal attention of a step's new tokens over a plain (bf16 or fp16) paged
// cache that already holds their keys and values (oscar_chunk_attention).
//
// Token j of a request's n, at position p = seq - n + j, sees the keys at
// positions max(0, p - window + 1) .. p:
//   o = sum_t exp(scale q.k_t - m) v_t / sum_t exp(scale q.k_t - m),
// m the running maximum: one pass over the keys, rescaling what is summed when
// the maximum is raised.  All heads that share a kv head are rows of one
// product, so a key is read once for (tokens x group) rows.
//
// The matrix unit works on transposed tiles: S^T = K Q^T (32 keys x 32 rows),
// then O^T += V^T P^T.  A lane owns one row throughout: it holds 16 of the
// tile's 32 scores of its row (the other half's lane the rest), its softmax is
// arithmetic in its own registers, and the score registers, rounded, are the
// next product's operand as they stand, because V's keys are taken in the order
// in which the score tile leaves them.  V^T comes from row-major V tiles by
// transposing LDS reads.
//
// The work is cut on the host into pieces (a 32-row tile of a request and kv
// head, or a wide one, over a range of keys) that fill the GPU; a row tile in
// several pieces leaves fp32 partials that a second launch joins.
//
// The matrix unit takes both operands in one type, so the weights are rounded to the
// cache's (off by 2^-8 of each at most in bf16, 2^-11 in fp16, as the output is by its
// own rounding) and summed as rounded: what remains is a mean with weights off by so
// much.  Scores, maxima, sums and partials are fp32.
//
// Times under "Measured" are of these kernels, with their spread between cards.
// Where two ways are set against each other, both were timed in turn on one card,
// with the rest of the kernels as it then was.
#include "plain_cache.h"
#include "row_span.h"

#include <algorithm>
#include <cstddef>
#include <cstring>
#include <functional>
#include <type_traits>
#include <utility>
#include <vector>

namespace oscar {
namespace {

constexpr int kTileKeys = 32;
constexpr int kTileRows = 32;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kCus = 256;
constexpr int32_t kMostKeys = 1 << 30;     // of a request, and rows: positions and windows add without overflow
constexpr float kNone = -3.0e38f;          // m before any key
// A row's m is its running maximum less Num<T>::kLift (both in units of a factor of
// 2), so that the largest weights lie between 2^kLift and 2^(kLift + kLazy): m is
// raised when a score exceeds it by kLift + kLazy.  bf16 has fp32's range, any place
// in it will do.  fp16 rounds weights below 2^-14 by steps of 2^-24; lifted by 2^7,
// up to half of its largest value, those are keys of less than 2^-21 of the heaviest
// one's weight, each off by 2^-32 of it at most.  (Without the lift 24000 keys of
// 2^-24.6 each counted half as much again.)
constexpr float kLazy = 8.f;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef uint16_t ushortx2 __attribute__((ext_vector_type(2)));
typedef uint16_t ushortx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) shortx4 lds_short4;

template <typename T>
struct Num;
template <>
struct Num<__bf16> {
  typedef bf16x8 V8;
  static __device__ __forceinline__ V8 round8(const float (&f)[8]) {
    // (settled here, in pairs: left to it, the compiler rounds value by value for
    // the comparisons that follow and again for the product)
    u32x4 w = __builtin_bit_cast(
        u32x4, __builtin_convertvector((floatx8{f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]}), V8));
    asm volatile("" : "+v"(w));
    return __builtin_bit_cast(V8, w);
  }
  static constexpr float kLift = 0.f;
  static constexpr float kMostWeight = 256.f;        // 2^(kLift + kLazy)
  static constexpr uint16_t kMostBits = 0x4380;      // its bits
  static constexpr uint16_t kInfBits = 0x7F80;
  static __device__ __forceinline__ floatx16 mfma(V8 a, V8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum8(V8 p, float l) {
    const bf16x2 one{(__bf16)1.f, (__bf16)1.f};
    l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 0, 1), one, l, false);
    l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 2, 3), one, l, false);
    l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 4, 5), one, l, false);
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 6, 7), one, l, false);
  }
};
template <>
struct Num<_Float16> {
  typedef half8 V8;
  static __device__ __forceinline__ V8 round8(const float (&f)[8]) {
    // (settled here, in pairs: left to it, the compiler rounds value by value for
    // the comparisons that follow and again for the product)
    u32x4 w = __builtin_bit_cast(
        u32x4, __builtin_convertvector((floatx8{f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]}), V8));
    asm volatile("" : "+v"(w));
    return __builtin_bit_cast(V8, w);
  }
  static constexpr float kLift = 7.f;
  static constexpr float kMostWeight = 32768.f;
  static constexpr uint16_t kMostBits = 0x7800;
  static constexpr uint16_t kInfBits = 0x7C00;
  static __device__ __forceinline__ floatx16 mfma(V8 a, V8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum8(V8 p, float l) {
    const half2v one{(_Float16)1.f, (_Float16)1.f};
    l = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 0, 1), one, l, false);
    l = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 2, 3), one, l, false);
    l = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 4, 5), one, l, false);
    return __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 6, 7), one, l, false);
  }
};

// A row tile over keys [key0, key1) of its request (key0 a multiple of 32).
struct Piece {
  int32_t token0;          // the request's first query token
  int32_t pos0;            // its position
  int32_t table_row;
  int32_t kv_head;
  int32_t row0, rows;      // of the request's (token, head) rows
  int32_t key0, key1;
  int32_t slot;            // first partial of 32 rows, -1: rows are finished here
  int32_t pad[3];
};
// 32 rows whose partials are slots slot0, slot0 + step, ...
struct Join {
  int32_t token0, kv_head, row0, rows, slot0, step, count, pad;
};
static_assert(sizeof(Piece) == 48 && sizeof(Join) == 32, "item sizes");

struct ChunkArgs {
  const uint8_t* q;
  uint8_t* out;
  int64_t q_token, q_head, out_token, out_head;      // bytes
  const uint8_t* k;
  const uint8_t* v;
  int64_t num_pages;
  uint32_t k_page, v_page;                           // bytes
  int32_t k_token, v_token, k_head, v_head;          // bytes
  const int32_t* table;
  int64_t table_stride;
  const Piece* pieces;
  const Join* joins;
  float* partials;         // slots of 32 rows: [32][D], then m[32], l[32]
  float scale_log2;
  int32_t group, block_size, window;
  int32_t narrow, wide;    // pieces, narrow ones first
  int32_t few_joins;       // joins of few partials come first
  FastDiv group_div, block_div;
};

// f(0), f(1), .. f(N - 1) with constants.
template <typename F, int... kI>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, kI...>) {
  (f(std::integral_constant<int, kI>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) { each_of(f, std::make_integer_sequence<int, N>{}); }

// x, opaque to the compiler: what is computed from it stays where it is written,
// instead of in registers through a loop.
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// x ^ kBits, computed where it is written.
template <int kBits>
__device__ __forceinline__ int xor_here(int x) {
  int y;
  asm volatile("v_xor_b32 %0, %1, %2" : "=v"(y) : "i"(kBits), "v"(x));
  return y;
}

// A product stays before what is written after it.
__device__ __forceinline__ void pin(floatx16& x) { asm volatile("" : "+v"(x)); }
// The instructions before this stay before those after it: a product's steps are
// written in the order in which they are to be issued.
__device__ __forceinline__ void keep_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}
// Every LDS and vector memory access of this wave done, then the workgroup's.
__device__ __forceinline__ void arrive_all() {
  __builtin_amdgcn_s_waitcnt(0x0070);       // vmcnt(0), lgkmcnt(0), expcnt left at its maximum
  asm volatile("s_barrier" ::: "memory");
}
__device__ __forceinline__ float max_halves(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return fmaxf(__int_as_float(s[0]), __int_as_float(s[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return __int_as_float(s[0]) + __int_as_float(s[1]);
}

// Tiles lie in LDS as rows of D values in 16-byte chunks, chunk c of key r at
// place c ^ swizzle(r), so that the reads below find their lanes' chunks on
// different banks: K's (32 keys, one chunk each) and V's (4 keys x 64 bytes a
// half wave).  Chunks move there by loads to LDS, whose lanes land one after
// the other: the lane picks the chunk that belongs at its place.
template <int D>
__device__ __forceinline__ int k_swizzle(int key) { return D >= 128 ? key & 15 : (key >> 1) & 7; }
template <int D>
__device__ __forceinline__ int v_swizzle(int key) { return D >= 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); }

// Pages of 64 groups of 16 keys from group `base` on, one a lane; -1: unmapped.
__device__ __forceinline__ int load_pages(const ChunkArgs& a, const Piece& p, int base, int lane) {
  const int key = 16 * (base + lane);
  int page = -1;
  if (key >= 0 && key < p.key1) {
    page = a.table[(int64_t)p.table_row * a.table_stride + fast_div((uint32_t)key, a.block_div)];
    page = page >= 0 && page < a.num_pages ? page : -1;
  }
  return page;
}

// Where a lane's 16 bytes lie in the first load of a run of keys: its key's row,
// and its chunk.  The loads that follow are some keys further on, and xor-ed with
// those keys' swizzle (their bits and the lane's are apart).
struct LanePlace {
  int row, chunk;          // bytes
};
template <int D, bool kV>
__device__ __forceinline__ LanePlace lane_place(const ChunkArgs& a, int lane) {
  constexpr int kLaneRow = D / 8;           // lanes of a row
  const int key = lane / kLaneRow, place = lane % kLaneRow;
  return LanePlace{key * (kV ? a.v_token : a.k_token),
                   16 * (place ^ (kV ? v_swizzle<D>(key) : k_swizzle<D>(key)))};
}

// How a load treats the caches: keys that other workgroups read too are kept,
// those that are read once (non-temporal) make no room for themselves: 8 users'
// token over 32K keys 49.1 us with this, 55.0 without.
constexpr int kKept = 0, kOnce = 2;

// Load kCount KB of consecutive keys from `key` on (inside one group of 16, at
// place in_page of `page`) to LDS: K or V rows of one kv head.  Keys past the
// piece's and unmapped pages arrive as zeros (records past the end).
template <int D, bool kV, int kCount, int kPolicy>
__device__ __forceinline__ void load_keys(const ChunkArgs& a, const Piece& p, int key, int key_in_tile, int page,
                                          int in_page, uint8_t* lds, const LanePlace& at) {
  constexpr int kStep = 512 / D;            // keys of a load
  const int stride = kV ? a.v_token : a.k_token;
  const int live = page < 0 ? 0 : min(16, p.key1 - key);
  const uint8_t* base = (kV ? a.v : a.k) + (int64_t)p.kv_head * (kV ? a.v_head : a.k_head) +
                        (uint64_t)(uint32_t)max(page, 0) * (kV ? a.v_page : a.k_page) + (uint32_t)(in_page * stride);
  const uint32_t records = live > 0 ? (uint32_t)((live - 1) * stride + 2 * D) : 0u;
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, records, 0x00020000);
#pragma unroll
  for (int n = 0; n < kCount; ++n) {
    const int first = key_in_tile + n * kStep;
    const int turn = 16 * (kV ? v_swizzle<D>(first) : k_swizzle<D>(first));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(lds + key_in_tile * 2 * D + n * 1024), 16,
                                             at.row + n * kStep * stride + (at.chunk ^ turn), 0, 0, kPolicy);
  }
}
// A key's place in its page.  (The high product is a vector instruction: back to
// a scalar, or the loads would loop over the descriptors of the lanes.)
__device__ __forceinline__ int place_in_page(const ChunkArgs& a, int key) {
  return __builtin_amdgcn_readfirstlane((int)fast_mod((uint32_t)key, a.block_div));
}

// A wave's 32 rows: queries, output sums, maximum and sum of weights.
template <typename T, int D>
struct RowState {
  typename Num<T>::V8 q[D / 16];
  floatx16 acc[D / 32];
  float m, l;              // l: of this half's keys
  int pos;                 // position of the lane's row
  int first, last;         // of the wave's rows
};

template <typename T, int D>
__device__ __forceinline__ void load_rows(const ChunkArgs& a, const Piece& p, int row0, int lane,
                                          RowState<T, D>& s) {
  const int end = p.row0 + p.rows - 1;
  const int row = min(row0 + (lane & 31), end);       // rows past the last repeat it and are not stored
  const int tok = (int)fast_div((uint32_t)row, a.group_div);
  const int head = row - tok * a.group + p.kv_head * a.group;
  const uint8_t* src = a.q + (int64_t)(p.token0 + tok) * a.q_token + (int64_t)head * a.q_head + 16 * (lane >> 5);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) s.q[i] = *reinterpret_cast<const typename Num<T>::V8*>(src + 32 * i);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) s.acc[i] = floatx16{};
  s.m = kNone;
  s.l = 0.f;
  s.pos = p.pos0 + tok;
  s.first = p.pos0 + (int)fast_div((uint32_t)min(row0, end), a.group_div);
  s.last = p.pos0 + (int)fast_div((uint32_t)min(row0 + kTileRows - 1, end), a.group_div);
}

// The first kCount scores a lane holds (register i: key 8 (i / 4) + 4 g + i % 4
// of the tile) that its row, at `pos`, does not see become -inf.  `unmapped`: bit
// h for keys 16h .. 16h + 15.
template <int kCount>
__device__ __forceinline__ void mask_scores(const ChunkArgs& a, floatx16& x, int key0, uint32_t unmapped, int lane,
                                            int pos) {
  const int hi = pos - key0 - 4 * (lane >> 5);
  const int lo = a.window == 0 ? INT32_MIN : hi - a.window;
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
    const int key = 8 * (i >> 2) + (i & 3);
    x[i] = key <= hi && key > lo && ((unmapped >> (i >> 3)) & 1u) == 0u ? x[i] : -__builtin_inff();
  }
}

// V^T operand of feature block b (in `place`, v_read ^ 64 b) and keys 8 (u / 4) + 4 g
// + u % 4 of the 16 that begin at vt.
template <typename T, int D>
__device__ __forceinline__ typename Num<T>::V8 v_operand_at(const uint8_t* vt, int place) {
  const uint8_t* at = vt + place;
  const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
  const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + 16 * D));
  return __builtin_bit_cast(typename Num<T>::V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Values that a row does not see must not reach it, and a weight of zero times an
// infinity or NaN would.  Tiles that every row sees whole need no care; in the
// others the wave looks over the values in LDS (kBytes) and, if some are not
// finite, makes them zeros there; what they do to the rows that do see them is
// added when the piece is done (add_special).  Waves that share a tile may do so
// at the same time: they write the same, and one at least has seen them.
template <typename T, int kBytes>
__device__ __forceinline__ bool take_out_special(uint8_t* vt, int lane) {
  ushortx8* const at = reinterpret_cast<ushortx8*>(vt) + lane;
  ushortx8 top{};
#pragma unroll
  for (int i = 0; i < kBytes / 1024; ++i) top = __builtin_elementwise_max(top, at[64 * i] & (uint16_t)0x7FFF);
  bool special = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) special = special || top[i] >= Num<T>::kInfBits;
  if (__builtin_expect(__ballot(special) == 0ull, 1)) return false;
#pragma unroll 1
  for (int i = 0; i < kBytes / 1024; ++i) {
    const ushortx8 u = at[64 * i];
    const ushortx8 below = Num<T>::kInfBits - (u & Num<T>::kInfBits);      // 0: not finite
    at[64 * i] = u & (0 - __builtin_elementwise_min(below, (ushortx8)(uint16_t)1));
  }
  return true;
}
// The values of a tile that are not finite, added to the sums of the rows that
// see them: what a positive weight makes of them.  Tiles that are whole and mapped
// had them in the product.
template <typename T, int D, int kKeys>
__device__ __forceinline__ void add_special(const ChunkArgs& a, const Piece& p, int key0, bool whole, int lane,
                                            RowState<T, D>& s) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  auto page_of = [&](int key) {
    const int page = a.table[(int64_t)p.table_row * a.table_stride + fast_div((uint32_t)key, a.block_div)];
    return page >= 0 && page < a.num_pages ? page : -1;
  };
  const int end = min(key0 + kKeys, p.key1);
  if (whole && page_of(key0) >= 0 && page_of(end - 1) >= 0) return;
  for (int key = key0; key < end; ++key) {
    const int page = page_of(key);
    if (page < 0) continue;
    const uint8_t* row = a.v + (int64_t)p.kv_head * a.v_head + (uint64_t)(uint32_t)page * a.v_page +
                         (uint64_t)fast_mod((uint32_t)key, a.block_div) * (uint32_t)a.v_token + 8 * (lane >> 5);
    const bool seen = key <= s.pos && (a.window == 0 || key > s.pos - a.window);
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const T4 x = *reinterpret_cast<const T4*>(row + 64 * b + 16 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = (float)x[i];
          s.acc[b][4 * j + i] += seen && !(fabsf(v) < __builtin_inff()) ? v : 0.f;
        }
        keep_order();                       // (few registers: this is rarely run)
      }
  }
}

// This lane's place in the reads of a K tile (key lane % 32, chunk 2 i + lane /
// 32 of k-step i) and of a V tile (keys 4 g + (lane % 16) / 4, 16 features of
// the lane's quarter).
template <int D>
__device__ __forceinline__ int k_read(int lane) {
  const int key = lane & 31;
  return key * 2 * D + 16 * ((lane >> 5) ^ k_swizzle<D>(key));
}
template <int D>
__device__ __forceinline__ int v_read(int lane) {
  const int key = 4 * (lane >> 5) + ((lane & 15) >> 2);
  return key * 2 * D + ((32 * ((lane >> 4) & 1) + 8 * (lane & 3)) ^ (16 * v_swizzle<D>(key)));
}

// Four values of a row, rounded.
template <typename T>
__device__ __forceinline__ void store4(uint8_t* at, floatx4 x) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<T4*>(at) = __builtin_convertvector(x, T4);
}

__device__ __forceinline__ uint8_t* out_row(const ChunkArgs& a, int token0, int kv_head, int row) {
  const int tok = (int)fast_div((uint32_t)row, a.group_div);
  const int head = row - tok * a.group + kv_head * a.group;
  return a.out + (int64_t)(token0 + tok) * a.out_token + (int64_t)head * a.out_head;
}

// ---------------------------------------------------------------- 32 rows
// One row tile, its keys shared out to four waves that walk their tiles on
// their own (no barrier until they combine): few rows, so memory bounds it, and
// what matters is loads in flight.  A wave's K and V tile each have one place
// in LDS; the next K tile is requested when the scores are done, the next V
// tile when its sums are, so that one or two tiles are always on their way.
// Tiles are 32 keys, or, beside wide pieces at D = 256, 16 (the upper half of the
// score tile is then the lower one's again and not used), so that two workgroups
// fit a CU's LDS; alone, few keys take longer with those (one token over 256 keys 8.7
// us, 8.0 with 32; 32 users' 4 tokens over 2K to 16K 55 with either).
// Measured: 8 users' token over 32K keys (D = 256) 48 us, 5.6 TB/s (a large copy
// moves 5.1, reading alone reaches 6.2 to 6.5); 32 users' 4 tokens over 2K to 16K 55
// us, 5.3 TB/s.  One user's over 1K takes 7.3 us and 3 of join: three memory round
// trips (piece, page, keys) and one for each of a wave's tiles.
constexpr int beside_keys(int d) { return d == 256 ? 16 : 32; }
constexpr int narrow_lds(int d, int keys) { return kWaves * 2 * keys * 2 * d + kWaves * 2 * kTileRows * 4; }

template <typename T, int D, int kKeys>
__device__ __forceinline__ void narrow_piece(const ChunkArgs& a, const Piece p, uint8_t* smem) {
  typedef typename Num<T>::V8 V8;
  constexpr int kHalves = kKeys / 16;
  constexpr int kTileBytes = kKeys * 2 * D;
  constexpr int kLoads = kTileBytes / 1024;
  constexpr int kBlocks = D / 32;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const int tiles = (p.key1 - p.key0 + kKeys - 1) / kKeys;
  const int first = p.key0 / kKeys + tiles * wave / kWaves;
  const int last = p.key0 / kKeys + tiles * (wave + 1) / kWaves;

  int page_base = kHalves * first;
  int pages = load_pages(a, p, page_base, lane);
  RowState<T, D> s;
  load_rows<T, D>(a, p, p.row0, lane, s);
  const int whole_from = a.window == 0 ? 0 : s.last - a.window + 1, whole_to = s.first - kKeys + 1;
  auto whole = [&](int key0) { return key0 >= whole_from && key0 <= whole_to; };
  bool special = false;                     // a tile that is not whole held values that are not finite

  const LanePlace k_place = lane_place<D, false>(a, lane), v_place = lane_place<D, true>(a, lane);
  auto page_of = [&](int t, int h) { return __builtin_amdgcn_readlane(pages, kHalves * t + h - page_base); };
  auto load_tile = [&](int t, auto v_tag, uint8_t* lds) {
    constexpr bool kV = decltype(v_tag)::value;
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
      load_keys<D, kV, kLoads / kHalves, kOnce>(a, p, t * kKeys + 16 * h, 16 * h, page_of(t, h),
                                         place_in_page(a, t * kKeys + 16 * h), lds, kV ? v_place : k_place);
  };
  const int k_addr = k_read<D>(lane & (32 + kKeys - 1)), v_addr = v_read<D>(lane);

  // One tile.  (The two places as parameters that do not alias: the compiler
  // then sees that a V read does not wait for the K tile that is on its way.)
  auto tile = [&](int t, uint8_t* __restrict__ kt, uint8_t* __restrict__ vt) __attribute__((always_inline)) {
    uint32_t unmapped = 0;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) unmapped |= page_of(t, h) < 0 ? 1u << h : 0u;
    const bool more = t + 1 < last;
    if (more && kHalves * (t + 1) - page_base >= 64) {
      page_base = kHalves * (t + 1);
      pages = load_pages(a, p, page_base, lane);
    }
    wait_vmcnt<kLoads>();                   // K is there, V on its way
    asm volatile("" ::: "memory");
    floatx16 x{};
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      x = Num<T>::mfma(*reinterpret_cast<const V8*>(kt + (k_addr ^ (32 * i))), s.q[i], x);
    asm volatile("" ::: "memory");
    if (more) load_tile(t + 1, std::false_type{}, kt);

    const int key0 = t * kKeys;
    const bool masked = !whole(key0) || unmapped != 0u;
    if (masked) mask_scores<8 * kHalves>(a, x, key0, unmapped, lane, s.pos);
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8 * kHalves; ++i) top = fmaxf(top, x[i]);
    top = max_halves(top) * a.scale_log2;
    const bool raise = top > s.m + (kLazy + Num<T>::kLift);
    if (__ballot(raise)) {
      const float m = raise ? top - Num<T>::kLift : s.m, f = __builtin_amdgcn_exp2f(s.m - m);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) s.acc[b] *= f;
      s.l *= f;
      s.m = m;
    }
    V8 w[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __builtin_amdgcn_exp2f(x[8 * h + i] * a.scale_log2 - s.m);
      w[h] = Num<T>::round8(f);
      s.l = Num<T>::sum8(w[h], s.l);
    }

    if (more) wait_vmcnt<kLoads>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    if (masked) special = take_out_special<T, kTileBytes>(vt, lane) || special;
    keep_order();
    each<kHalves * kBlocks>([&](auto step) {
      constexpr int h = decltype(step)::value / kBlocks, b = decltype(step)::value % kBlocks;
      s.acc[b] = Num<T>::mfma(v_operand_at<T, D>(vt + h * 32 * D, v_addr ^ (64 * b)), w[h], s.acc[b]);
      if constexpr (b % 4 == 3 || b == kBlocks - 1) keep_order();
    });
    asm volatile("" ::: "memory");
    if (more) load_tile(t + 1, std::true_type{}, vt);
  };
  uint8_t* const kt = smem + wave * 2 * kTileBytes;
  if (first < last) {
    load_tile(first, std::false_type{}, kt);
    __builtin_amdgcn_sched_barrier(0);      // (the waits count K's loads before V's)
    load_tile(first, std::true_type{}, kt + kTileBytes);
  }
  for (int t = first; t < last; ++t) tile(t, kt, kt + kTileBytes);
  if (__builtin_expect(special, 0))
    for (int t = first; t < last; ++t) add_special<T, D, kKeys>(a, p, t * kKeys, whole(t * kKeys), lane, s);

  // Combine: the waves' sums through LDS, D / kRounds features at a time (16-byte
  // pieces, the row xor-ed in).
  constexpr int kRounds = 32 / kKeys, kPart = D / kRounds;
  float* const sums = reinterpret_cast<float*>(smem);
  float* const ml = sums + kWaves * kTileRows * kPart;          // [wave][m | l][32]
  s.l = sum_halves(s.l);
  const int row = lane & 31;
#pragma unroll
  for (int round = 0; round < kRounds; ++round) {
    arrive_all();
    if (row < p.rows) {
#pragma unroll
      for (int b = 0; b < kPart / 32; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int piece = 8 * b + 2 * i + (lane >> 5);
          const floatx16& acc = s.acc[round * kPart / 32 + b];
          *reinterpret_cast<floatx4*>(sums + (wave * kTileRows + row) * kPart + 4 * (piece ^ (row & 15))) =
              floatx4{acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]};
        }
      ml[wave * 64 + (lane >> 5) * 32 + row] = lane < 32 ? s.m : s.l;
    }
    __syncthreads();
    // a thread to four features of some rows, kBatch of them at once
    constexpr int kAcross = kThreads / (kPart / 4), kBatch = kAcross >= 16 ? 1 : 16 / kAcross;
    const int piece = tid % (kPart / 4), feature = round * kPart + 4 * piece;
    for (int r0 = tid / (kPart / 4); r0 < p.rows; r0 += kAcross * kBatch) {
      float m[kBatch], l[kBatch];
      floatx4 o[kBatch];
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int r = min(r0 + n * kAcross, p.rows - 1);
        float wm[kWaves], wl[kWaves];
        floatx4 x[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          wm[w] = ml[w * 64 + r];
          wl[w] = ml[w * 64 + 32 + r];
          x[w] = *reinterpret_cast<const floatx4*>(sums + (w * kTileRows + r) * kPart + 4 * (piece ^ (r & 15)));
        }
        m[n] = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
        l[n] = 0.f;
        o[n] = floatx4{};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(wm[w] - m[n]);
          l[n] += f * wl[w];
          o[n] += f * x[w];
        }
      }
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int r = r0 + n * kAcross;
        if (r >= p.rows) break;
        if (p.slot < 0) {
          const float inv = l[n] == 0.f ? 0.f : 1.f / l[n];
          store4<T>(out_row(a, p.token0, p.kv_head, p.row0 + r) + 2 * feature, o[n] * inv);
        } else {
          float* part = a.partials + (int64_t)p.slot * (kTileRows * (D + 2));
          *reinterpret_cast<floatx4*>(part + r * D + feature) = o[n];
          if (feature == 0) {
            part[kTileRows * D + r] = m[n];
            part[kTileRows * D + kTileRows + r] = l[n];
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------- 128 rows
// A wide row tile: four waves of 32 rows each, over stages of keys in LDS that
// all four read, two stages in turn: while one is computed, the next is on its
// way.  A wave does a tile's products and softmax one after the other; the
// matrix unit is kept busy by the waves of the other workgroups on the CU, which
// no barrier ties to this one.
// Two workgroups of four waves fill the registers at D = 256 (64 of queries, 128 of
// sums a lane), so the order in which a tile's products and reads are issued is
// written out: the compiler's own spills registers to memory.
// What bounds it: the matrix unit together with the vector instructions of the
// softmax (and, at D = 64, those alone: 16 exponentials a lane against 8 products),
// at the clock the power limit leaves (1.6 GHz in the longest cases).  Measured:
// D = 256, 6 heads on one, 9256 tokens over 15360 keys 960 to 1120 us, 1.0 to 1.19
// PFLOP/s; D = 128, 32 on 8, 8192 over 8192 1440 to 1550 us, 1.06 to 1.14; D = 64, 16
// on 4, 8192 over 8192 410 to 435 us, 0.95 to 1.0 (a large bf16 matrix product: 1.34
// to 1.38).
constexpr int kWideRows = 32 * kWaves;
constexpr int kWideWgs = 2;                                      // workgroups a CU
constexpr int stage_tiles(int d) { return d == 256 ? 1 : 2; }    // 32-key tiles of a stage

constexpr int wide_lds(int d) { return 2 * 2 * stage_tiles(d) * kTileKeys * 2 * d; }

template <typename T, int D>
__device__ __forceinline__ void wide_piece(const ChunkArgs& a, const Piece p, uint8_t* smem) {
  typedef typename Num<T>::V8 V8;
  constexpr int kTiles = stage_tiles(D);
  constexpr int kTileBytes = kTileKeys * 2 * D;
  constexpr int kStageBytes = 2 * kTiles * kTileBytes;           // K tiles, then V tiles
  constexpr int kLoads = kTiles * kTileBytes / 1024 / kWaves;    // of a stage's K, a wave
  constexpr int kKeys = kTiles * kTileKeys / kWaves;             // that it loads: inside a group of 16
  constexpr int kSteps = D / 16, kBlocks = D / 32, kPv = 2 * kBlocks;
  constexpr int kAheadK = D == 128 ? 6 : 4, kAheadV = D == 256 ? 3 : D == 128 ? 6 : 4;     // operands read ahead
  constexpr bool kKeepAddresses = D <= 128;      // of the operand reads in registers (D = 256 has none left)
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles = (p.key1 - p.key0 + kTileKeys - 1) / kTileKeys;
  const int group0 = p.key0 / 16;

  int page_base = group0;
  int pages = load_pages(a, p, page_base, lane);
  RowState<T, D> s;
  load_rows<T, D>(a, p, p.row0 + kTileRows * wave, lane, s);

  LanePlace k_place = lane_place<D, false>(a, lane), v_place = lane_place<D, true>(a, lane);
  const int k_addr = k_read<D>(lane), v_addr = v_read<D>(lane);
  // A stage's keys of this wave: their page and place in it (found with K's
  // request, V's are the same), and which groups of 16 keys are unmapped.
  int page = 0, in_page = place_in_page(a, p.key0 + kKeys * wave);
  const int advance = place_in_page(a, kTiles * kTileKeys);
  uint32_t gone_next = 0;
  auto request_k = [&](int stage, uint8_t* to) __attribute__((always_inline)) {
    const int group = group0 + 2 * kTiles * stage;
    if (group - page_base >= 64) {
      page_base = group;
      pages = load_pages(a, p, page_base, opaque(lane));
    }
    const int at = group - page_base;
    gone_next = 0;
#pragma unroll
    for (int h = 0; h < 2 * kTiles; ++h) {
      const int g = __builtin_amdgcn_readlane(pages, at + h);
      gone_next |= g < 0 ? 1u << h : 0u;
      page = h == 0 || kKeys * wave >= 16 * h ? g : page;
    }
    if (stage > 0) {
      in_page += advance;
      in_page -= in_page >= a.block_size ? a.block_size : 0;
    }
    load_keys<D, false, kLoads, kKept>(a, p, p.key0 + kTiles * kTileKeys * stage + kKeys * wave, kKeys * wave, page,
                                       in_page, to, k_place);
  };
  auto request_v = [&](int stage, uint8_t* to) __attribute__((always_inline)) {
    load_keys<D, true, kLoads, kKept>(a, p, p.key0 + kTiles * kTileKeys * stage + kKeys * wave, kKeys * wave, page,
                                      in_page, to + kTiles * kTileBytes, v_place);
  };
  // The operands' places: steps i and i + kSteps / 2 of the first product, and blocks
  // b and b + kBlocks / 2 of the second, lie a constant apart at D = 256 (there the
  // xor-ed bits are below it), so they are taken in turn and share a register.
  int k_place_now, v_place_now;
  auto k_step = [](int j) { return kKeepAddresses ? j : (j >> 1) + (j & 1) * (kSteps / 2); };
  auto v_block = [](int j) { return kKeepAddresses ? j : (j >> 1) + (j & 1) * (kBlocks / 2); };
  auto k_operand = [&](const uint8_t* kt, auto step) {
    constexpr int j = decltype(step)::value;
    if constexpr (kKeepAddresses) return *reinterpret_cast<const V8*>(kt + (k_addr ^ (32 * j)));
    if constexpr (j % 2 == 0) k_place_now = xor_here<16 * j>(k_addr);
    return *reinterpret_cast<const V8*>(kt + k_place_now + j % 2 * D);
  };
  auto v_operand = [&](const uint8_t* vt, auto step) {
    constexpr int h = decltype(step)::value / kBlocks, j = decltype(step)::value % kBlocks;
    if constexpr (kKeepAddresses) return v_operand_at<T, D>(vt + h * 32 * D, v_addr ^ (64 * j));
    if constexpr (j % 2 == 0) v_place_now = xor_here<32 * j>(v_addr);
    return v_operand_at<T, D>(vt + h * 32 * D + j % 2 * D, v_place_now);
  };
  // Rows that do not see the whole of a tile lose what they do not see.  (Asked of
  // the workgroup's rows together: its waves share the tiles.)
  const int pos0 = p.pos0 + (int)fast_div((uint32_t)p.row0, a.group_div);
  const int pos1 = p.pos0 + (int)fast_div((uint32_t)(p.row0 + p.rows - 1), a.group_div);
  const int whole_from = a.window == 0 ? 0 : pos1 - a.window + 1, whole_to = pos0 - kTileKeys + 1;
  auto whole = [&](int key0) { return key0 >= whole_from && key0 <= whole_to; };
  bool special = false;                     // this wave found values that are not finite in such a tile
  auto weight = [&](float x) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.scale_log2, -s.m)); };
  auto weigh = [&](const floatx16& x, V8 (&w)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = weight(x[8 * h + i]);
      w[h] = Num<T>::round8(f);
      __builtin_amdgcn_sched_barrier(0);    // (eight at a time: registers)
    }
  };
  // Whether some weight is above the most (or no number) shows in the tile's sum of
  // weights at D = 128; at the other sizes the sums are added up beside the second
  // product and the weights asked (from the sum / from the weights: 8 prompts of 300
  // over 500, D = 128, 45.7 / 50.8 us; 6000 + 1501 tokens in a window, D = 64, 49 /
  // 45.5; 9256 over 15360, D = 256, 1127 / 1104).
  constexpr bool kSumFirst = D == 128;
  auto sum = [](const V8 (&w)[2]) { return Num<T>::sum8(w[0], 0.f) + Num<T>::sum8(w[1], 0.f); };
  // Positive numbers compare as their bits do, so this takes nine operations for a
  // tile, where the maximum of the scores takes one for each.
  auto beyond = [&](const V8 (&w)[2]) {
    const ushortx8 u = __builtin_elementwise_max(__builtin_bit_cast(ushortx8, w[0]), __builtin_bit_cast(ushortx8, w[1]));
    const ushortx2 top = __builtin_elementwise_max(
        __builtin_elementwise_max(__builtin_shufflevector(u, u, 0, 1), __builtin_shufflevector(u, u, 2, 3)),
        __builtin_elementwise_max(__builtin_shufflevector(u, u, 4, 5), __builtin_shufflevector(u, u, 6, 7)));
    const ushortx2 most{Num<T>::kMostBits, Num<T>::kMostBits};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(top, most)) != 0u;
  };
  // Raises the running maximum to that of the tile's scores where a weight, or their
  // sum, was too large (always so for the first keys of a row), and rescales the sums.
  // A row is asked for its heaviest weight just as it was rounded: other rows stay as
  // they are, so what becomes of a row does not depend on its neighbours.  (Asked for
  // its score, one whose weight rounds to the most would be raised beside a heavier
  // neighbour, but not by itself.)
  auto raise = [&](const floatx16& x, float l) __attribute__((always_inline)) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
    top = max_halves(top);
    const float heaviest = (float)(T)weight(top);
    top *= a.scale_log2;
    const bool over = kSumFirst ? !(max_halves(l) <= Num<T>::kMostWeight) && top - Num<T>::kLift > s.m
                                : heaviest > Num<T>::kMostWeight;
    const float m = over ? top - Num<T>::kLift : s.m, f = __builtin_amdgcn_exp2f(s.m - m);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) s.acc[b] *= f;
    s.l *= f;
    s.m = m;
  };

  // One tile; `requests(i)` goes out beside step i of its first product.
  auto tile = [&](const uint8_t* __restrict__ kt, uint8_t* __restrict__ vt, int key0, uint32_t gone,
                  auto&& requests) __attribute__((always_inline)) {
    if constexpr (!kKeepAddresses) {
      k_place = LanePlace{opaque(k_place.row), opaque(k_place.chunk)};
      v_place = LanePlace{opaque(v_place.row), opaque(v_place.chunk)};
    }
    // S^T = K Q^T
    V8 k[kAheadK];
    each<kAheadK>([&](auto step) { k[decltype(step)::value] = k_operand(kt, step); });
    keep_order();
    __builtin_amdgcn_s_setprio(1);
    floatx16 x;
    each<kSteps>([&](auto step) {
      constexpr int i = decltype(step)::value;
      x = Num<T>::mfma(k[i % kAheadK], s.q[k_step(i)], i == 0 ? floatx16{} : x);
      pin(x);
      if constexpr (i + kAheadK < kSteps) k[i % kAheadK] = k_operand(kt, std::integral_constant<int, i + kAheadK>{});
      keep_order();
      requests(i);
      keep_order();
    });
    __builtin_amdgcn_s_setprio(0);
    if (__builtin_expect(!whole(key0) || gone != 0u, 0)) {
      mask_scores<16>(a, x, key0, gone, lane, s.pos);
      special = take_out_special<T, kTileBytes>(vt, lane) || special;
    }
    V8 v[kAheadV];
    each<kAheadV>([&](auto step) { v[decltype(step)::value] = v_operand(vt, step); });
    V8 w[2];
    weigh(x, w);
    float l = kSumFirst ? sum(w) : 0.f;
    if (__ballot(kSumFirst ? !(l <= Num<T>::kMostWeight) : beyond(w))) {
      raise(x, l);
      weigh(x, w);
      if constexpr (kSumFirst) l = sum(w);
    }
    if constexpr (kSumFirst) s.l += l;
    keep_order();
    __builtin_amdgcn_s_setprio(1);
    // O^T += V^T P^T
    each<kPv>([&](auto step) {
      constexpr int i = decltype(step)::value, h = i / kBlocks, b = v_block(i % kBlocks);
      s.acc[b] = Num<T>::mfma(v[i % kAheadV], w[h], s.acc[b]);
      pin(s.acc[b]);
      if constexpr (i + kAheadV < kPv) v[i % kAheadV] = v_operand(vt, std::integral_constant<int, i + kAheadV>{});
      if constexpr (b == 0 && !kSumFirst) s.l = Num<T>::sum8(w[h], s.l);
      keep_order();
    });
    __builtin_amdgcn_s_setprio(0);
  };

  request_k(0, smem);
  request_v(0, smem);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {        // the queries are in registers before the sums take theirs
    u32x4 q = __builtin_bit_cast(u32x4, s.q[i]);
    asm volatile("" : "+v"(q));
    s.q[i] = __builtin_bit_cast(V8, q);
  }
  keep_order();
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) s.acc[b] = floatx16{};
  int stage = 0;
  auto run = [&](uint8_t* __restrict__ now, uint8_t* __restrict__ next) __attribute__((always_inline)) {
    wait_vmcnt<0>();                        // this stage is there,
    asm volatile("s_barrier" ::: "memory"); // and nobody reads the place of the next one
    const uint32_t gone = gone_next;
    const int key0 = p.key0 + kTiles * kTileKeys * stage;
    ++stage;
#pragma unroll
    for (int u = 0; u < kTiles; ++u) {
      if (u > 0 && kTiles * (stage - 1) + u >= tiles) break;
      tile(now + u * kTileBytes, now + (kTiles + u) * kTileBytes, key0 + u * kTileKeys, (gone >> (2 * u)) & 3u,
           [&](int i) __attribute__((always_inline)) {
             if (u == 0 && i == 0) request_k(stage, next);
             if (u == 0 && i == (kSteps > 4 ? 3 : 1)) request_v(stage, next);
           });
    }
  };
  // (two stages a turn, so that their places are constants of the reads)
  while (kTiles * stage < tiles) {
    run(smem, smem + kStageBytes);
    if (kTiles * stage >= tiles) break;
    run(smem + kStageBytes, smem);
  }
  arrive_all();                             // (loads to LDS that nobody waits for)
  if (lane == 0) reinterpret_cast<int*>(smem)[wave] = special;
  arrive_all();
  const u32x4 found = *reinterpret_cast<const u32x4*>(smem);
  if (__builtin_expect(__builtin_amdgcn_readfirstlane(found[0] | found[1] | found[2] | found[3]) != 0, 0))
    for (int key0 = p.key0; key0 < p.key1; key0 += kTileKeys)
      add_special<T, D, kTileKeys>(a, p, key0, whole(key0), lane, s);

  const float l = sum_halves(s.l);
  const int at = kTileRows * wave + (lane & 31);
  if (at >= p.rows) return;
  if (p.slot < 0) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint8_t* o = out_row(a, p.token0, p.kv_head, p.row0 + at) + 8 * (lane >> 5);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4<T>(o + 64 * b + 16 * i,
                  floatx4{s.acc[b][4 * i], s.acc[b][4 * i + 1], s.acc[b][4 * i + 2], s.acc[b][4 * i + 3]} * inv);
  } else {
    float* part = a.partials + (int64_t)(p.slot + wave) * (kTileRows * (D + 2));
    float* o = part + (lane & 31) * D + 4 * (lane >> 5);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<floatx4*>(o + 32 * b + 8 * i) =
            floatx4{s.acc[b][4 * i], s.acc[b][4 * i + 1], s.acc[b][4 * i + 2], s.acc[b][4 * i + 3]};
    if (lane < 32) {
      part[kTileRows * D + (lane & 31)] = s.m;
      part[kTileRows * D + kTileRows + (lane & 31)] = l;
    }
  }
}

// ---------------------------------------------------------------- kernels
// (LDS of fixed size: its place is then known when addresses are computed, which in
// the wide tiles' steps is one addition an operand less: D = 256, 9256 tokens over
// 15360 1190 -> 1130 us.)
constexpr int narrow_wgs(int d) { return 256 / d; }             // workgroups a CU
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

// ---------------------------------------------------------------- join
// The partials of cut row tiles.  A 32-row group of few partials (kFewParts): a
// thread to four features of a row, 256 to a workgroup, all partials at once.  Of
// more: a workgroup to 64 features of a row, 16 threads across the features and
// 16 across the partials, whose sums meet in LDS.  (Few up to 8: 2048 tokens beside
// 16 users' 4, D = 256, 180 us, up to 4 203, up to 16 183.)  The partials' bytes bound
// it (512 wide pieces of D = 128: 43 MB, 9.7 us), or, where there is little, latency:
// 2.3 to 5 us.
constexpr int kFewParts = 8;

template <typename T, int D, int kParts>
__device__ __forceinline__ void join_few(const ChunkArgs& a, const Join j, int block) {
  const int i = block * 256 + (int)threadIdx.x, row = i / (D / 4), feature = 4 * (i % (D / 4));
  if (row >= j.rows) return;
  const float* const first = a.partials + (int64_t)j.slot0 * (kTileRows * (D + 2));
  float m[kParts], l[kParts], top = kNone;
  floatx4 x[kParts];
#pragma unroll
  for (int s = 0; s < kParts; ++s) {        // (the last one again for those that are not there: no load waits)
    const float* at = first + (int64_t)(min(s, j.count - 1) * j.step) * (kTileRows * (D + 2));
    m[s] = at[kTileRows * D + row];
    l[s] = at[kTileRows * D + kTileRows + row];
    x[s] = *reinterpret_cast<const floatx4*>(at + row * D + feature);
  }
#pragma unroll
  for (int s = 0; s < kParts; ++s) top = fmaxf(top, m[s]);
  floatx4 o{};
  float sum = 0.f;
#pragma unroll
  for (int s = 0; s < kParts; ++s)
    if (s < j.count) {
      const float w = __builtin_amdgcn_exp2f(m[s] - top);
      sum += w * l[s];
      o += w * x[s];
    }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  store4<T>(out_row(a, j.token0, j.kv_head, j.row0 + row) + 2 * feature, o * inv);
}

template <typename T, int D>
__device__ __forceinline__ void join_many(const ChunkArgs& a, const Join j, int row, int part64) {
  const int tid = (int)threadIdx.x, feature = 64 * part64 + 4 * (tid & 15), part = tid >> 4;
  __shared__ float red[16][64 + 4];
  __shared__ float red_m[16], red_l[16];
  auto slot = [&](int i) { return a.partials + (int64_t)(j.slot0 + i * j.step) * (kTileRows * (D + 2)); };
  float m = kNone;
  for (int i = part; i < j.count; i += 16) m = fmaxf(m, slot(i)[kTileRows * D + row]);
  floatx4 o{};
  float l = 0.f;
  for (int i = part; i < j.count; i += 16) {
    const float* s = slot(i);
    const float w = __builtin_amdgcn_exp2f(s[kTileRows * D + row] - m);
    l += w * s[kTileRows * D + kTileRows + row];
    o += w * *reinterpret_cast<const floatx4*>(s + row * D + feature);
  }
  *reinterpret_cast<floatx4*>(&red[part][4 * (tid & 15)]) = o;
  if ((tid & 15) == 0) {
    red_m[part] = m;
    red_l[part] = l;
  }
  __syncthreads();
  if (tid >= 16) return;
  float top = red_m[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) top = fmaxf(top, red_m[i]);
  floatx4 sum{};
  float lsum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float w = __builtin_amdgcn_exp2f(red_m[i] - top);
    lsum += w * red_l[i];
    sum += w * *reinterpret_cast<const floatx4*>(&red[i][4 * tid]);
  }
  const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
  store4<T>(out_row(a, j.token0, j.kv_head, j.row0 + row) + 2 * feature, sum * inv);
}

// Groups of few partials first, D / 32 workgroups each; then 32 x D / 64 a group.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(ChunkArgs a) {
  constexpr int kFewBlocks = D / 32, kManyBlocks = kTileRows * D / 64;
  const int block = (int)blockIdx.x, few = a.few_joins * kFewBlocks;
  if (block < few) {
    const Join j = a.joins[block / kFewBlocks];
    if (j.count <= 2) join_few<T, D, 2>(a, j, block % kFewBlocks);
    else if (j.count <= 4) join_few<T, D, 4>(a, j, block % kFewBlocks);
    else join_few<T, D, kFewParts>(a, j, block % kFewBlocks);
    return;
  }
  const int many = (block - few) / kManyBlocks, at = (block - few) % kManyBlocks;
  const Join j = a.joins[a.few_joins + many];
  if (at / (D / 64) < j.rows) join_many<T, D>(a, j, at / (D / 64), at % (D / 64));
}

// ---------------------------------------------------------------- the plan
struct Plan {
  std::vector<Piece> narrow, wide;
  std::vector<Join> joins;
  int32_t slots = 0;
};

struct RowTile {
  Piece piece;
  int32_t tiles;           // of 32 keys
};

// The row tiles of a request, `rows` rows each, with the keys that they see.
void row_tiles(int32_t token0, int32_t n, int32_t seq, int32_t table_row, int32_t group, int32_t kv_heads,
               int32_t window, int32_t rows, std::vector<RowTile>& out) {
  const int32_t all = n * group;
  for (int32_t r = 0; r < all; r += rows) {
    Piece p{};
    p.token0 = token0;
    p.pos0 = seq - n;
    p.table_row = table_row;
    p.row0 = r;
    p.rows = std::min(rows, all - r);
    p.slot = -1;
    const int32_t lo = window > 0 ? std::max(0, p.pos0 + r / group - window + 1) : 0;
    p.key0 = lo / kTileKeys * kTileKeys;
    p.key1 = p.pos0 + (r + p.rows - 1) / group + 1;
    for (int32_t h = 0; h < kv_heads; ++h) {
      p.kv_head = h;
      out.push_back(RowTile{p, (p.key1 - p.key0 + kTileKeys - 1) / kTileKeys});
    }
  }
}

// A row tile in n pieces of equal length, but for a key tile.
void cut(const RowTile& x, int32_t n, Plan& plan, std::vector<Piece>& out) {
  if (n <= 1) {
    out.push_back(x.piece);
    return;
  }
  const int32_t groups = (x.piece.rows + kTileRows - 1) / kTileRows;
  for (int32_t g = 0; g < groups; ++g)
    plan.joins.push_back(Join{x.piece.token0, x.piece.kv_head, x.piece.row0 + g * kTileRows,
                              std::min(kTileRows, x.piece.rows - g * kTileRows), plan.slots + g, groups, n, 0});
  for (int32_t s = 0; s < n; ++s) {
    Piece p = x.piece;
    p.key0 = x.piece.key0 + kTileKeys * (int32_t)((int64_t)x.tiles * s / n);
    p.key1 = std::min<int32_t>(x.piece.key1, x.piece.key0 + kTileKeys * (int32_t)((int64_t)x.tiles * (s + 1) / n));
    p.slot = plan.slots;
    plan.slots += groups;
    out.push_back(p);
  }
}

int32_t pieces_of(const RowTile& x, int64_t per) { return (int32_t)((x.tiles + per - 1) / per); }

// Narrow tiles: the fewest key tiles a piece, one number for all row tiles, with which
// there is a piece a CU at most, or, where that leaves the longest piece a seventh
// above the mean, as many pieces as reside at once (D = 128: 8 users' 4 tokens over
// 4000 keys, 8 kv heads, a piece a CU 27.3 us, two 28.7, 4 users' over 2048 10.4, 12.8;
// 24 users' over 100 to 16200 a piece a CU 166 us, two 140).  Where the longest row
// tile is short, all stay whole, and there is no second launch: one token of one user
// over 256 keys, D = 256, whole 7.9 us of GPU time, cut 8.3 (over 512: 10.9, 8.3); D =
// 128, 8 kv heads, over 512 whole 7.2, cut 7.1 and 6.2 against 10.6 where the host
// launches (over 1024: 11.1, 7.0).
// Beside wide tiles that take at least two thirds of the reading's time (`beside`, in
// their units, of which a narrow tile's 128 D bytes at 5.2 TB/s are 1/160), two narrow
// workgroups to three CUs (16 users over 8000 keys beside two prompts, D = 256: 37 to
// 45 us, two a CU 43 to 55; 12 over 2000 beside 512 tokens, D = 128: 30, 35); where the
// reading takes longer, two a CU (16 over 8000 beside two prompts, D = 128: 107 us, two
// to three CUs 128).
// So row tiles are cut only as far as there are fewer of them than that many pieces:
// where there are as many or more, all stay whole, in the order of the requests.  That
// is right for even lengths, and for ragged ones (256 users of 100 to 8000 keys, D =
// 256, 190 us, 5.2 TB/s), but one request that is far longer than the others is then
// read by one workgroup (300 users of 1000 keys and one of 131072 2.2 ms, where the
// bytes take 0.09), and by a few where there are just fewer (250 and one: 0.39 ms).
void plan_narrow(const std::vector<RowTile>& rows, int32_t head_size, double beside, Plan& plan) {
  int64_t total = 0;
  int32_t most = 0;
  for (const RowTile& x : rows) {
    total += x.tiles;
    most = std::max(most, x.tiles);
  }
  const int32_t uncut = head_size == 256 ? 8 : 16;
  auto fit = [&](int64_t resident) {
    int64_t per = std::max<int64_t>(kWaves, (total + resident - 1) / resident);
    auto count = [&](int64_t t) {
      int64_t c = 0;
      for (const RowTile& x : rows) c += pieces_of(x, t);
      return c;
    };
    if ((int64_t)rows.size() >= resident || most <= uncut) per = std::max<int64_t>(per, most);
    // (The count falls as pieces get longer.  Step by step the search took 5 ms for 250
    // short rows beside 2^20 keys, and 17 s beside 2^30.)
    for (int64_t high = std::max<int64_t>(per, most); per < high;) {
      const int64_t mid = (per + high) / 2;
      if (count(mid) > resident) per = mid + 1;
      else high = mid;
    }
    return per;
  };
  int64_t per = fit(beside == 0. ? kCus : total > 240 * beside ? 2 * kCus : 2 * kCus / 3);
  if (beside == 0. && (rows.size() >= kCus || 100 * per * kCus > 115 * total))
    per = fit((int64_t)kCus * narrow_wgs(head_size));
  for (const RowTile& x : rows) cut(x, pieces_of(x, per), plan, plan.narrow);
}

// Wide tiles.  Workgroups take pieces as they come free, two to a CU.  Row tiles
// are left whole or cut in pieces of at most so many key tiles, whichever is
// estimated to end first.  In units of a key tile's time on a busy CU (D = 256 0.97
// us, 128 0.47, 64 0.27): a piece costs 4 beside its tiles, one of a cut row tile 15
// (its partials are written and read again: the same at any D, as both go with D);
// a workgroup alone on its CU takes 1.07, 1.45 or 1.5 units a tile; the join is a
// launch of 5 us; cut pieces end a tenth later than their sum, as they are not dealt
// out as is assumed here.  Measured, whole / cut, us:
//   D = 256, 6 heads: 9256 tokens over 15360 1081 / 1143, 4096 over 28672 1061 /
//   711, 3001 alone 98 / 54, 1024 alone 40 / 28, 77 over 20011 578 / 33;
//   D = 128, 32 heads: 1024 over 4096 111 / 88, 8 prompts of 300 over 500 50 / 70;
//   D = 64, 16 heads: 8192 over 8192 412 / 425, 1024 over 1024 37 / 23, 6000 + 1501
//   tokens in a window of 1024 45 / 59.
// Cuts are tried while their number times all row tiles stays within kMostPieces, also
// where only some row tiles are long enough to be cut: beside many short prompts a
// chunk over a long cache stays whole (8 prompts of 512 beside 64 tokens over 32768,
// D = 128, 640 us, where the keys take 43).
// Returns the estimate.
constexpr int32_t kPieceCost = 4, kCutCost = 15, kLeastPiece = 8, kMostPieces = 2048;
double plan_wide(const std::vector<RowTile>& rows, int32_t head_size, Plan& plan) {
  int32_t most = 0;
  for (const RowTile& x : rows) most = std::max(most, x.tiles);
  const double alone = head_size == 256 ? 1.07 : head_size == 128 ? 1.45 : 1.5;
  const double join = head_size == 256 ? 5.0 : head_size == 128 ? 11.0 : 18.0;
  // In pieces of at most `per` key tiles, dealt out to the CUs longest first, there
  // and back.
  std::vector<int32_t> count;               // of pieces, by cost
  std::vector<int64_t> load(kCus);
  auto parted = [&](int32_t per) {
    count.assign(per + kCutCost + 1, 0);
    bool cuts = false;
    for (const RowTile& x : rows) {
      const int32_t n = pieces_of(x, per);
      cuts = cuts || n > 1;
      count[(x.tiles + n - 1) / n + (n > 1 ? kCutCost : kPieceCost)] += n;
    }
    std::fill(load.begin(), load.end(), 0);
    int64_t dealt = 0, longest = 0;
    for (int32_t cost = (int32_t)count.size() - 1; cost > 0; --cost)
      for (int32_t n = count[cost]; n > 0; --n, ++dealt) {
        const int64_t at = dealt % kCus;
        load[dealt / kCus % 2 ? kCus - 1 - at : at] += cost;
        longest = std::max<int64_t>(longest, cost);
      }
    const double busiest = (double)*std::max_element(load.begin(), load.end());
    return std::max(cuts ? 1.1 * busiest : busiest, alone * longest) + (cuts ? join : 0.);
  };
  int32_t per = most;
  double best = parted(most);
  for (int32_t parts = 2; (size_t)parts * rows.size() <= kMostPieces; parts += 1 + parts / 8) {
    const int32_t at_most = (most + parts - 1) / parts;
    if (at_most < kLeastPiece) break;
    const double t = parted(at_most);
    if (t < best) {
      best = t;
      per = at_most;
    }
  }
  for (const RowTile& x : rows) cut(x, pieces_of(x, per), plan, plan.wide);
  std::stable_sort(plan.wide.begin(), plan.wide.end(),
                   [](const Piece& x, const Piece& y) { return x.key1 - x.key0 > y.key1 - y.key0; });
  // The first two rounds of workgroups share CUs in order: the longest pieces,
  // shortest first, meet the next ones, longest first.
  std::reverse(plan.wide.begin(), plan.wide.begin() + (std::ptrdiff_t)std::min<size_t>(kCus, plan.wide.size()));
  return best;
}

void make_plan(const int32_t* qsl, const int32_t* seqs, int32_t num_requests, int32_t group, int32_t kv_heads,
               int32_t head_size, int32_t window, Plan& plan) {
  // Up to 32 rows a request is narrow (28 rows of 16 users over 1000 keys, D = 128: 20.4
  // us, as wide tiles 24.2; 30 of 8 users over 16000, D = 256, 31.1, 30.1), from 33 on
  // wide, where narrow tiles would read its keys twice (48 rows, the same: 24.7 us, as
  // narrow 23.2; 32.2, 36.1; 32 users over 4000 32.5, 49.6).
  std::vector<RowTile> narrow, wide;
  for (int32_t i = 0; i < num_requests; ++i) {
    const int32_t n = qsl[i + 1] - qsl[i];
    if (n * (int64_t)group <= kTileRows)
      row_tiles(qsl[i], n, seqs[i], i, group, kv_heads, window, kTileRows, narrow);
    else
      row_tiles(qsl[i], n, seqs[i], i, group, kv_heads, window, kWideRows, wide);
  }
  const double beside = wide.empty() ? 0. : plan_wide(wide, head_size, plan);
  if (!narrow.empty()) plan_narrow(narrow, head_size, beside, plan);
  std::stable_partition(plan.joins.begin(), plan.joins.end(), [](const Join& j) { return j.count <= kFewParts; });
}

template <typename T, int D>
int launch(const ChunkArgs& a, const oscar_chunk_step& step, hipStream_t stream) {
  static_assert(kWideWgs * mixed_lds(D) <= 160 * 1024 && narrow_wgs(D) * narrow_lds(D, kTileKeys) <= 160 * 1024,
                "the workgroups of a CU must fit its 160 KiB of LDS");
  void (*const kernels[3])(ChunkArgs) = {&narrow_kernel<T, D>, &wide_kernel<T, D>, &mixed_kernel<T, D>};
  const int which = step.wide == 0 ? 0 : step.narrow == 0 ? 1 : 2;
  kernels[which]<<<step.narrow + step.wide, kThreads, 0, stream>>>(a);
  const int64_t blocks = (int64_t)step.few_joins * (D / 32) + (int64_t)(step.joins - step.few_joins) * (kTileRows * D / 64);
  if (blocks > INT32_MAX) return kErrInvalidArgument;
  if (blocks > 0) join_kernel<T, D><<<(uint32_t)blocks, 256, 0, stream>>>(a);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
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

extern "C" int oscar_chunk_plan(const int32_t* query_start_loc, const int32_t* seq_lens, int32_t num_requests,
                                int32_t num_heads, int32_t window, const oscar_plain_cache* cache, void* items,
                                size_t items_size, oscar_chunk_step* step) {
  using namespace oscar;
  const int status = check_chunk_cache(cache);
  if (status != kOk) return status;
  if (step == nullptr || num_requests < 0 || (num_requests > 0 && (query_start_loc == nullptr || seq_lens == nullptr)) ||
      num_heads < 1 || num_heads % cache->num_kv_heads || num_heads > (1 << 16) || window < 0)
    return kErrInvalidArgument;
  const int32_t group = num_heads / cache->num_kv_heads;
  int32_t pages = 0;
  for (int32_t i = 0; i < num_requests; ++i) {
    const int64_t n = (int64_t)query_start_loc[i + 1] - query_start_loc[i];
    if (query_start_loc[i] < 0 || n < 0 || seq_lens[i] < n || n * group > kMostKeys ||
        seq_lens[i] > kMostKeys)
      return kErrInvalidArgument;
    if (n > 0) pages = std::max(pages, (seq_lens[i] - 1) / cache->block_size + 1);
  }
  try {
    Plan plan;
    make_plan(query_start_loc, seq_lens, num_requests, group, cache->num_kv_heads, cache->head_size, window, plan);
    const size_t narrow = plan.narrow.size() * sizeof(Piece), wide = plan.wide.size() * sizeof(Piece);
    const size_t joins = plan.joins.size() * sizeof(Join);
    if (plan.narrow.size() + plan.wide.size() > INT32_MAX || plan.joins.size() > INT32_MAX) return kErrInvalidArgument;
    step->num_requests = num_requests;
    step->num_tokens = num_requests > 0 ? query_start_loc[num_requests] : 0;
    step->num_heads = num_heads;
    step->num_kv_heads = cache->num_kv_heads;
    step->head_size = cache->head_size;
    step->block_size = cache->block_size;
    step->window = std::min(window, kMostKeys);
    step->table_cols = pages;
    step->narrow = (int32_t)plan.narrow.size();
    step->wide = (int32_t)plan.wide.size();
    step->joins = (int32_t)plan.joins.size();
    step->few_joins = (int32_t)std::count_if(plan.joins.begin(), plan.joins.end(),
                                             [](const Join& j) { return j.count <= kFewParts; });
    step->items_size = (int64_t)(narrow + wide + joins);
    step->workspace_size = (int64_t)plan.slots * kTileRows * (cache->head_size + 2) * 4;
    if (items == nullptr) return kOk;
    if (items_size < narrow + wide + joins) return kErrWorkspaceTooSmall;
    uint8_t* to = static_cast<uint8_t*>(items);
    if (narrow > 0) std::memcpy(to, plan.narrow.data(), narrow);
    if (wide > 0) std::memcpy(to + narrow, plan.wide.data(), wide);
    if (joins > 0) std::memcpy(to + narrow + wide, plan.joins.data(), joins);
  } catch (...) {
    return kErrInvalidArgument;
  }
  return kOk;
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
  if (step->narrow < 0 || step->wide < 0 || step->few_joins < 0 || step->joins < step->few_joins)
    return kErrInvalidArgument;
  if (step->narrow + step->wide == 0) return kOk;
  if (items == nullptr || block_table == nullptr || query->data == nullptr || out->data == nullptr ||
      block_table_stride < step->table_cols)
    return kErrInvalidArgument;
  if ((int64_t)workspace_size < step->workspace_size || (step->workspace_size > 0 && workspace == nullptr))
    return kErrWorkspaceTooSmall;
  ChunkArgs a{};
  a.q = static_cast<const uint8_t*>(query->data);
  a.out = static_cast<uint8_t*>(out->data);
  if (step->num_tokens > 1) {               // (a stride between rows of which there is one means nothing)
    a.q_token = 2 * query->token_stride;
    a.out_token = 2 * out->token_stride;
  }
  if (step->num_heads > 1) {
    a.q_head = 2 * query->head_stride;
    a.out_head = 2 * out->head_stride;
  }
  if (((uintptr_t)query->data | (uintptr_t)out->data | (uintptr_t)workspace | (uintptr_t)items) % 16 ||
      (a.q_token | a.q_head | a.out_token | a.out_head) % 16 ||
      std::min({a.q_token, a.q_head, a.out_token, a.out_head}) < 0)
    return kErrUnsupportedGeometry;
  // (a row is read by the workgroup that writes it, or by a launch before the one that does)
  const RowSpan from{(uint64_t)(uintptr_t)a.q, a.q_token, a.q_head, step->num_tokens, step->num_heads,
                     2 * cache->head_size};
  const RowSpan to{(uint64_t)(uintptr_t)a.out, a.out_token, a.out_head, step->num_tokens, step->num_heads,
                   2 * cache->head_size};
  if (!same_rows(from, to) && !rows_apart(from, to)) return kErrOverlap;
  a.k = static_cast<const uint8_t*>(cache->k);
  a.v = static_cast<const uint8_t*>(cache->v);
  a.k_page = (uint32_t)cache->k_stride_page;
  a.v_page = (uint32_t)cache->v_stride_page;
  a.num_pages = cache->num_pages;
  a.k_token = (int32_t)cache->k_stride_token;
  a.v_token = (int32_t)cache->v_stride_token;
  a.k_head = (int32_t)cache->k_stride_head;
  a.v_head = (int32_t)cache->v_stride_head;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.pieces = static_cast<const Piece*>(items);
  a.narrow = step->narrow;
  a.wide = step->wide;
  a.few_joins = step->few_joins;
  a.joins = reinterpret_cast<const Join*>(a.pieces + step->narrow + step->wide);
  a.partials = static_cast<float*>(workspace);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.group = step->num_heads / cache->num_kv_heads;
  a.block_size = cache->block_size;
  a.window = step->window;
  a.group_div = make_fast_div((uint32_t)a.group);
  a.block_div = make_fast_div((uint32_t)a.block_size);
  return cache->dtype == OSCAR_BF16 ? launch_sized<__bf16>(cache->head_size, a, *step, stream)
                                    : launch_sized<_Float16>(cache->head_size, a, *step, stream);
}
