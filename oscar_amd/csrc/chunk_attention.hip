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
#include "plain_cache.h"

#include <algorithm>
#include <cstring>
#include <functional>
#include <type_traits>
#include <vector>

namespace oscar {
namespace {

constexpr int kTileKeys = 32;
constexpr int kTileRows = 32;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kCus = 256;
constexpr int32_t kMostKeys = 1 << 30;     // of a request, and rows: positions and windows add without overflow
constexpr float kNone = -3.0e38f;          // running maximum before any key
constexpr float kLazy = 8.f;               // a maximum is raised when a score exceeds it by 2^8

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) shortx4 lds_short4;

template <typename T>
struct Num;
template <>
struct Num<__bf16> {
  typedef bf16x8 V8;
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
  int64_t k_page, v_page, num_pages;
  int32_t k_token, v_token, k_head, v_head;          // bytes
  const int32_t* table;
  int64_t table_stride;
  const Piece* pieces;
  const Join* joins;
  float* partials;         // slots of 32 rows: [32][D], then m[32], l[32]
  float scale_log2;
  int32_t group, block_size, window;
  int32_t wide0;           // first piece of the wide kernel
  FastDiv group_div, block_div;
};

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}
// Every LDS and vector memory access of this wave done, then the workgroup's.
__device__ __forceinline__ void arrive_all() {
  __builtin_amdgcn_s_waitcnt(0x0070);       // vmcnt(0), lgkmcnt(0), expcnt left at its maximum
  asm volatile("s_barrier" ::: "memory");
}
__device__ __forceinline__ float other_half(float x) {       // lane ^ 32's
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return (threadIdx.x & 32) != 0 ? __int_as_float(s[0]) : __int_as_float(s[1]);
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

// Load kCount KB of consecutive keys from `key` on (inside one group of 16)
// to LDS: K or V rows of one kv head.  Keys past the piece's and unmapped pages
// arrive as zeros (records past the end).
template <int D, bool kV, int kCount>
__device__ __forceinline__ void load_keys(const ChunkArgs& a, const Piece& p, int key, int key_in_tile, int page,
                                          uint8_t* lds, int lane) {
  constexpr int kLaneRow = D / 8;           // lanes of a row
  constexpr int kStep = 512 / D;            // keys of a load
  const int stride = kV ? a.v_token : a.k_token;
  const uint8_t* base = kV ? a.v : a.k;
  const int in_page = (int)fast_mod((uint32_t)key, a.block_div);
  const int live = page < 0 ? 0 : min(16, p.key1 - key);
  base += (int64_t)max(page, 0) * (kV ? a.v_page : a.k_page) + (int64_t)in_page * stride +
          (int64_t)p.kv_head * (kV ? a.v_head : a.k_head);
  const uint32_t records = live > 0 ? (uint32_t)((live - 1) * stride + 2 * D) : 0u;
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, records, 0x00020000);
  const int lane_key = lane / kLaneRow, place = lane % kLaneRow;
#pragma unroll
  for (int n = 0; n < kCount; ++n) {
    const int r = n * kStep + lane_key;     // key of this lane, from `key` on
    const int chunk = place ^ (kV ? v_swizzle<D>(key_in_tile + r) : k_swizzle<D>(key_in_tile + r));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(lds + key_in_tile * 2 * D + n * 1024), 16,
                                             r * stride + 16 * chunk, 0, 0, 0);
  }
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

// S^T = K Q^T of one tile.
template <typename T, int D>
__device__ __forceinline__ floatx16 scores(const uint8_t* kt, int k_addr, const RowState<T, D>& s) {
  floatx16 x{};
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    x = Num<T>::mfma(*reinterpret_cast<const typename Num<T>::V8*>(kt + (k_addr ^ (32 * i))), s.q[i], x);
  return x;
}

// Weights of one tile: exp2(score - m), rounded to T for the product and summed
// as rounded, so that the output stays a mean of the values.  `unmapped`: bit h
// for keys 16h .. 16h + 15.
template <typename T, int D>
__device__ __forceinline__ void weights(const ChunkArgs& a, floatx16& x, int key0, uint32_t unmapped, int lane,
                                        RowState<T, D>& s, typename Num<T>::V8 (&p)[2]) {
  const bool whole = key0 + kTileKeys - 1 <= s.first && (a.window == 0 || key0 > s.last - a.window) && unmapped == 0u;
  if (!whole) {
    const int g4 = 4 * (lane >> 5);
    const int hi = s.pos - key0 - g4;       // register i holds key 8 (i / 4) + 4 g + i % 4
    const int lo = a.window == 0 ? INT32_MIN : hi - a.window;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = 8 * (i >> 2) + (i & 3);
      const bool seen = key <= hi && key > lo && ((unmapped >> (i >> 3)) & 1u) == 0u;
      x[i] = seen ? x[i] : -__builtin_inff();
    }
  }
  float top = x[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
  top = max_halves(top) * a.scale_log2;
  const bool raise = top > s.m + kLazy;
  if (__ballot(raise)) {
    const float m = raise ? top : s.m;
    const float alpha = __builtin_amdgcn_exp2f(s.m - m);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) s.acc[i] *= alpha;
    s.l *= alpha;
    s.m = m;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] * a.scale_log2 - s.m);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    floatx8 w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = x[8 * h + i];
    p[h] = __builtin_convertvector(w, typename Num<T>::V8);
    s.l = Num<T>::sum8(p[h], s.l);
  }
}

// O^T += V^T P^T of one tile: feature block b of keys 16 h + 8 (u / 4) + 4 g + u % 4.
template <typename T, int D>
__device__ __forceinline__ void values(const uint8_t* vt, int v_addr, const typename Num<T>::V8 (&p)[2],
                                       RowState<T, D>& s) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int b = 0; b < D / 32; ++b) {
      const uint8_t* at = vt + (v_addr ^ (64 * b)) + h * 32 * D;
      const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
      const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + 16 * D));
      const shortx8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      s.acc[b] = Num<T>::mfma(__builtin_bit_cast(typename Num<T>::V8, v), p[h], s.acc[b]);
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
// tile when its sums are, so that one or two tiles (32 D .. 128 D bytes a wave)
// are always on their way.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 1) void narrow_kernel(ChunkArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int kTileBytes = kTileKeys * 2 * D;
  constexpr int kLoads = D / 16;            // of a tile
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Piece p = a.pieces[blockIdx.x];
  uint8_t* kt = smem + wave * 2 * kTileBytes;
  uint8_t* vt = kt + kTileBytes;

  const int tiles = (p.key1 - p.key0 + kTileKeys - 1) / kTileKeys;
  const int first = p.key0 / kTileKeys + tiles * wave / kWaves;
  const int last = p.key0 / kTileKeys + tiles * (wave + 1) / kWaves;

  int page_base = 2 * first;
  int pages = load_pages(a, p, page_base, lane);
  RowState<T, D> s;
  load_rows<T, D>(a, p, p.row0, lane, s);

  auto page_of = [&](int t, int h) { return __builtin_amdgcn_readlane(pages, 2 * t + h - page_base); };
  auto load_tile = [&](int t, auto v_tag, uint8_t* lds) {
    constexpr bool kV = decltype(v_tag)::value;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      load_keys<D, kV, kLoads / 2>(a, p, t * kTileKeys + 16 * h, 16 * h, page_of(t, h), lds, lane);
  };
  const int k_addr = k_read<D>(lane), v_addr = v_read<D>(lane);

  if (first < last) {
    load_tile(first, std::false_type{}, kt);
    __builtin_amdgcn_sched_barrier(0);      // (the waits below count K's loads before V's)
    load_tile(first, std::true_type{}, vt);
  }
  // One tile.  (The two places as parameters that do not alias: the compiler
  // then sees that a V read does not wait for the K tile that is on its way.)
  auto tile = [&](int t, uint8_t* __restrict__ kt, uint8_t* __restrict__ vt) __attribute__((always_inline)) {
    const uint32_t unmapped = (page_of(t, 0) < 0 ? 1u : 0u) | (page_of(t, 1) < 0 ? 2u : 0u);
    const bool more = t + 1 < last;
    if (more && 2 * (t + 1) - page_base >= 64) {
      page_base = 2 * (t + 1);
      pages = load_pages(a, p, page_base, lane);
    }
    wait_vmcnt<kLoads>();                   // K is there, V on its way
    asm volatile("" ::: "memory");
    floatx16 x = scores<T, D>(kt, k_addr, s);
    asm volatile("" ::: "memory");
    if (more) load_tile(t + 1, std::false_type{}, kt);
    typename Num<T>::V8 w[2];
    weights<T, D>(a, x, t * kTileKeys, unmapped, lane, s, w);
    if (more) wait_vmcnt<kLoads>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    values<T, D>(vt, v_addr, w, s);
    asm volatile("" ::: "memory");
    if (more) load_tile(t + 1, std::true_type{}, vt);
  };
  for (int t = first; t < last; ++t) tile(t, kt, vt);

  // Combine: every wave's sums to LDS (16-byte pieces, the row xor-ed in).
  float* sums = reinterpret_cast<float*>(smem);
  float* ml = sums + kWaves * kTileRows * D;          // [wave][m | l][32]
  s.l = sum_halves(s.l);
  arrive_all();
  const int row = lane & 31;
  if (row < p.rows) {
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int piece = 8 * b + 2 * i + (lane >> 5);
        *reinterpret_cast<floatx4*>(sums + (wave * kTileRows + row) * D + 4 * (piece ^ (row & 15))) =
            floatx4{s.acc[b][4 * i], s.acc[b][4 * i + 1], s.acc[b][4 * i + 2], s.acc[b][4 * i + 3]};
      }
    ml[wave * 64 + (lane >> 5) * 32 + row] = lane < 32 ? s.m : s.l;
  }
  __syncthreads();
  for (int i = tid; i < p.rows * (D / 4); i += kThreads) {
    const int r = i / (D / 4), piece = i % (D / 4);
    float m = ml[r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, ml[w * 64 + r]);
    floatx4 o{};
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml[w * 64 + r] - m);
      l += f * ml[w * 64 + 32 + r];
      o += f * *reinterpret_cast<const floatx4*>(sums + (w * kTileRows + r) * D + 4 * (piece ^ (r & 15)));
    }
    if (p.slot < 0) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      store4<T>(out_row(a, p.token0, p.kv_head, p.row0 + r) + 8 * piece, o * inv);
    } else {
      float* part = a.partials + (int64_t)p.slot * (kTileRows * (D + 2));
      *reinterpret_cast<floatx4*>(part + r * D + 4 * piece) = o;
      if (piece == 0) {
        part[kTileRows * D + r] = m;
        part[kTileRows * D + kTileRows + r] = l;
      }
    }
  }
}

// ---------------------------------------------------------------- 256 rows
// A wide row tile: kW waves of kR times 32 rows each, over tiles of 32 keys that
// all of them read from LDS.  The scores of a tile are computed one tile ahead,
// so that products and softmax overlap inside a wave: iteration t runs
//   A:  S(t + 1) = K Q^T        beside the weights of the tile's first 16 keys,
//   B1: O += V^T P^T, 16 keys   beside the weights of the other 16,
//   B2: O += V^T P^T, 16 keys   beside the maximum of S(t + 1),
// each step of a product followed by its share of the arithmetic (the order is
// the schedule: scheduling barriers keep it).  K and V tiles come through rings
// of four places, requested two iterations ahead; one barrier an iteration, in
// the middle of B, where the K tile just used and the V tile before this one
// are given up.
constexpr int kWideRows = 256;
constexpr int kRing = 4;

template <int D>
constexpr int wide_lds() { return 2 * kRing * kTileKeys * 2 * D; }

template <typename T, int D, int kR, int kW, int kWgs>
__global__ __launch_bounds__(64 * kW, kW * kWgs / 4) void wide_kernel(ChunkArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  typedef typename Num<T>::V8 V8;
  constexpr int kTileBytes = kTileKeys * 2 * D;
  constexpr int kLoads = kTileBytes / 1024 / kW;       // of a tile and wave
  constexpr int kKeys = kTileKeys / kW;                // keys of a tile that a wave loads
  constexpr int kSteps = D / 16, kBlocks = D / 32;
  constexpr int kAhead = D == 256 ? 2 : 4;
  static_assert(kLoads * 1024 * kW == kTileBytes && kR * kW * 32 == kWideRows, "whole kilobytes a wave");
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Piece p = a.pieces[a.wide0 + blockIdx.x];
  uint8_t* const kring = smem;
  uint8_t* const vring = smem + kRing * kTileBytes;
  const int tiles = (p.key1 - p.key0 + kTileKeys - 1) / kTileKeys;
  const int group0 = p.key0 / 16;

  int page_base = group0;
  int pages = load_pages(a, p, page_base, lane);
  RowState<T, D> s[kR];
#pragma unroll
  for (int r = 0; r < kR; ++r) load_rows<T, D>(a, p, p.row0 + 32 * (kR * wave + r), lane, s[r]);
  const int first = s[0].first, last = s[kR - 1].last;

  // Tile u's page of this wave's keys (kept until its V is requested, two tiles
  // later), and which halves of the tiles from the last requested one back are
  // unmapped, two bits each.
  int page_next = 0, page_after = 0;
  uint32_t unmapped = 0;
  auto request_k = [&](int u) {
    const int g = group0 + 2 * u - page_base;
    if (g >= 64) {
      page_base += g;
      pages = load_pages(a, p, page_base, lane);
    }
    const int at = group0 + 2 * u - page_base;
    const int lo = __builtin_amdgcn_readlane(pages, at), hi = __builtin_amdgcn_readlane(pages, at + 1);
    const int page = kKeys * wave < 16 ? lo : hi;
    unmapped = (unmapped << 2) | (lo < 0 ? 1u : 0u) | (hi < 0 ? 2u : 0u);
    load_keys<D, false, kLoads>(a, p, p.key0 + u * kTileKeys + kKeys * wave, kKeys * wave, page,
                                kring + (u % kRing) * kTileBytes, lane);
    return page;
  };
  auto request_v = [&](int u, int page) {
    load_keys<D, true, kLoads>(a, p, p.key0 + u * kTileKeys + kKeys * wave, kKeys * wave, page,
                               vring + (u % kRing) * kTileBytes, lane);
  };
  // (the waits below count these in this order)
  const int p0 = request_k(0);
  __builtin_amdgcn_sched_barrier(0);
  const int p1 = request_k(1);
  page_next = request_k(2);
  request_v(0, p0);
  __builtin_amdgcn_sched_barrier(0);
  page_after = request_k(3);
  request_v(1, p1);
  __builtin_amdgcn_sched_barrier(0);

  const int k_addr = k_read<D>(lane), v_addr = v_read<D>(lane);
  auto k_operand = [&](const uint8_t* kt, int i) {
    return *reinterpret_cast<const V8*>(kt + (k_addr ^ (32 * i)));
  };
  auto v_operand = [&](const uint8_t* vt, int h, int b) {
    const uint8_t* at = vt + (v_addr ^ (64 * b)) + h * 32 * D;
    const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
    const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + 16 * D));
    return __builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // The running maxima, raised where a tile's scores ask for it.
  auto raise_max = [&](float (&top)[kR]) {
    bool raise[kR], any = false;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      top[r] = max_halves(top[r]) * a.scale_log2;
      raise[r] = top[r] > s[r].m + kLazy;
      any = any || raise[r];
    }
    if (__ballot(any)) {
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const float m = raise[r] ? top[r] : s[r].m, f = __builtin_amdgcn_exp2f(s[r].m - m);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) s[r].acc[b] *= f;
        s[r].l *= f;
        s[r].m = m;
      }
    }
  };
  // Rows that do not see the whole of tile u lose what they do not see.
  auto mask_tile = [&](floatx16 (&x)[kR], int u, uint32_t gone) {
    const int key0 = p.key0 + u * kTileKeys;
    if (key0 + kTileKeys - 1 <= first && (a.window == 0 || key0 > last - a.window) && gone == 0u) return;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int hi = s[r].pos - key0 - 4 * (lane >> 5);
      const int lo = a.window == 0 ? INT32_MIN : hi - a.window;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 8 * (i >> 2) + (i & 3);
        x[r][i] = key <= hi && key > lo && ((gone >> (i >> 3)) & 1u) == 0u ? x[r][i] : -__builtin_inff();
      }
    }
  };

  // ---- first scores ----
  floatx16 xa[kR], xb[kR];
  wait_vmcnt<5 * kLoads>();                 // K(0) is there
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int r = 0; r < kR; ++r) xa[r] = floatx16{};
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const V8 k = k_operand(kring, i);
#pragma unroll
    for (int r = 0; r < kR; ++r) xa[r] = Num<T>::mfma(k, s[r].q[i], xa[r]);
  }
  mask_tile(xa, 0, (unmapped >> 6) & 3u);
  float top[kR];
#pragma unroll
  for (int r = 0; r < kR; ++r) {
    top[r] = xa[r][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top[r] = fmaxf(top[r], xa[r][i]);
  }
  raise_max(top);
  wait_vmcnt<2 * kLoads>();                 // K(1), K(2), V(0) are there
  asm volatile("s_barrier" ::: "memory");
  {
    const int page = request_k(4);
    request_v(2, page_next);
    page_next = page_after;
    page_after = page;
  }

  // One iteration: tile t's scores are in x, tile t + 1's come to y.
  auto iterate = [&](int t, floatx16 (&x)[kR], floatx16 (&y)[kR], uint8_t* __restrict__ kr,
                     uint8_t* __restrict__ vr) __attribute__((always_inline)) {
    const uint8_t* kt = kr + ((t + 1) % kRing) * kTileBytes;
    const uint8_t* vt = vr + (t % kRing) * kTileBytes;
    V8 w[kR][2];                            // [rows][key half]
    auto weight = [&](int e) {
#pragma unroll
      for (int r = 0; r < kR; ++r) x[r][e] = __builtin_amdgcn_exp2f(x[r][e] * a.scale_log2 - s[r].m);
    };
    auto round = [&](int h) {
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        floatx8 f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = x[r][8 * h + i];
        w[r][h] = __builtin_convertvector(f, V8);
        s[r].l = Num<T>::sum8(w[r][h], s[r].l);
      }
    };
    // A
    V8 k[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) k[i] = k_operand(kt, i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int r = 0; r < kR; ++r) y[r] = Num<T>::mfma(k[i % kAhead], s[r].q[i], i == 0 ? floatx16{} : y[r]);
      if (i + kAhead < kSteps) k[i % kAhead] = k_operand(kt, i + kAhead);
#pragma unroll
      for (int e = i * 8 / kSteps; e < (i + 1) * 8 / kSteps; ++e) weight(e);
      __builtin_amdgcn_sched_barrier(0);
    }
    V8 v[kAhead];
    constexpr int kPv = 2 * kBlocks;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = v_operand(vt, i / kBlocks, i % kBlocks);
    round(0);
    __builtin_amdgcn_sched_barrier(0);
    mask_tile(y, t + 1, (unmapped >> 6) & 3u);
    // B1, B2
    float top[kR];
#pragma unroll
    for (int i = 0; i < kPv; ++i) {
      const int h = i / kBlocks, b = i % kBlocks;
      if (i == kBlocks) {
        round(1);
        wait_vmcnt<2 * kLoads>();           // K(t + 2), V(t + 1) are there
        asm volatile("s_barrier" ::: "memory");
        const int page = request_k(t + 5);
        request_v(t + 3, page_next);
        page_next = page_after;
        page_after = page;
      }
#pragma unroll
      for (int r = 0; r < kR; ++r) s[r].acc[b] = Num<T>::mfma(v[i % kAhead], w[r][h], s[r].acc[b]);
      if (i + kAhead < kPv) v[i % kAhead] = v_operand(vt, (i + kAhead) / kBlocks, (i + kAhead) % kBlocks);
      if (h == 0) {
#pragma unroll
        for (int e = 8 + b * 8 / kBlocks; e < 8 + (b + 1) * 8 / kBlocks; ++e) weight(e);
      } else {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          if (b == 0) top[r] = y[r][0];
#pragma unroll
          for (int e = b * 16 / kBlocks; e < (b + 1) * 16 / kBlocks; ++e) top[r] = fmaxf(top[r], y[r][e]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    raise_max(top);
  };
  for (int t = 0; t < tiles; t += 2) {
    iterate(t, xa, xb, kring, vring);
    if (t + 1 < tiles) iterate(t + 1, xb, xa, kring, vring);
  }
  arrive_all();                             // (loads to LDS that nobody waits for)

#pragma unroll
  for (int r = 0; r < kR; ++r) {
    const float l = sum_halves(s[r].l);
    const int at = 32 * (kR * wave + r) + (lane & 31);
    if (at >= p.rows) continue;
    if (p.slot < 0) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint8_t* o = out_row(a, p.token0, p.kv_head, p.row0 + at) + 8 * (lane >> 5);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          store4<T>(o + 64 * b + 16 * i, floatx4{s[r].acc[b][4 * i], s[r].acc[b][4 * i + 1], s[r].acc[b][4 * i + 2],
                                                 s[r].acc[b][4 * i + 3]} * inv);
    } else {
      float* part = a.partials + (int64_t)(p.slot + kR * wave + r) * (kTileRows * (D + 2));
      float* o = part + (lane & 31) * D + 4 * (lane >> 5);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<floatx4*>(o + 32 * b + 8 * i) =
              floatx4{s[r].acc[b][4 * i], s[r].acc[b][4 * i + 1], s[r].acc[b][4 * i + 2], s[r].acc[b][4 * i + 3]};
      if (lane < 32) {
        part[kTileRows * D + (lane & 31)] = s[r].m;
        part[kTileRows * D + kTileRows + (lane & 31)] = l;
      }
    }
  }
}

// ---------------------------------------------------------------- join
// One row and 64 of its features a workgroup: 16 threads across the features,
// 16 across the partials.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(ChunkArgs a) {
  const Join j = a.joins[blockIdx.x];
  const int row = (int)blockIdx.y;
  if (row >= j.rows) return;
  const int tid = (int)threadIdx.x, feature = 64 * (int)blockIdx.z + 4 * (tid & 15), part = tid >> 4;
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

// A row tile in n pieces of equal parts of its keys.
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

// Narrow tiles: the fewest key tiles a piece with which the pieces fit the
// workgroups that are resident at once.
void plan_narrow(const std::vector<RowTile>& rows, int32_t head_size, Plan& plan) {
  int64_t total = 0;
  int32_t most = 0;
  for (const RowTile& x : rows) {
    total += x.tiles;
    most = std::max(most, x.tiles);
  }
  const int64_t resident = (int64_t)kCus * (256 / head_size);
  int64_t per = std::max<int64_t>(kWaves, (total + resident - 1) / resident);
  auto count = [&](int64_t t) {
    int64_t c = 0;
    for (const RowTile& x : rows) c += pieces_of(x, t);
    return c;
  };
  if ((int64_t)rows.size() >= resident) per = std::max<int64_t>(per, most);
  while (per < most && count(per) > resident) ++per;
  for (const RowTile& x : rows) cut(x, pieces_of(x, per), plan, plan.narrow);
}

// Wide tiles: workgroups take pieces as they come free, the longest first.  Of
// a few piece lengths the one whose pieces, dealt out to the workgroups that
// are resident at once, end first.
constexpr int32_t kPieceCost = 5;          // of a piece beside its tiles, in tiles' time
void plan_wide(const std::vector<RowTile>& rows, int32_t head_size, Plan& plan) {
  int64_t total = 0;
  int32_t most = 0;
  for (const RowTile& x : rows) {
    total += x.tiles;
    most = std::max(most, x.tiles);
  }
  const int64_t resident = (int64_t)kCus * (head_size == 64 ? 2 : 1);
  int64_t best = most, best_end = INT64_MAX;
  std::vector<int32_t> length;
  std::vector<int64_t> load;
  for (int64_t k = 0; k <= 4; ++k) {
    const int64_t per = k == 0 ? most : std::max<int64_t>(8, (total + resident * k - 1) / (resident * k));
    if (per > most || (k > 0 && (int64_t)rows.size() > 4 * resident)) continue;
    length.clear();
    for (const RowTile& x : rows) {
      const int32_t n = pieces_of(x, per);
      for (int32_t i = 0; i < n; ++i) length.push_back((x.tiles + n - 1) / n + kPieceCost * (n > 1 ? 2 : 1));
    }
    std::sort(length.begin(), length.end(), std::greater<int32_t>());
    load.assign((size_t)resident, 0);
    for (size_t i = 0; i < length.size(); ++i) {
      const size_t at = i % (size_t)resident;
      load[(i / (size_t)resident) % 2 ? (size_t)resident - 1 - at : at] += length[i];
    }
    const int64_t end = *std::max_element(load.begin(), load.end());
    if (end < best_end) {
      best_end = end;
      best = per;
    }
  }
  for (const RowTile& x : rows) cut(x, pieces_of(x, best), plan, plan.wide);
  std::stable_sort(plan.wide.begin(), plan.wide.end(),
                   [](const Piece& x, const Piece& y) { return x.key1 - x.key0 > y.key1 - y.key0; });
}

void make_plan(const int32_t* qsl, const int32_t* seqs, int32_t num_requests, int32_t group, int32_t kv_heads,
               int32_t head_size, int32_t window, Plan& plan) {
  std::vector<RowTile> narrow, wide;
  for (int32_t i = 0; i < num_requests; ++i) {
    const int32_t n = qsl[i + 1] - qsl[i];
    if (n * (int64_t)group <= kTileRows)
      row_tiles(qsl[i], n, seqs[i], i, group, kv_heads, window, kTileRows, narrow);
    else
      row_tiles(qsl[i], n, seqs[i], i, group, kv_heads, window, kWideRows, wide);
  }
  if (!narrow.empty()) plan_narrow(narrow, head_size, plan);
  if (!wide.empty()) plan_wide(wide, head_size, plan);
}

constexpr size_t narrow_lds(int d) { return (size_t)kWaves * kTileRows * d * 4 + kWaves * 64 * 4; }

template <typename T, int D>
int launch(const ChunkArgs& a, const oscar_chunk_step& step, hipStream_t stream) {
  if (step.narrow > 0) {
    static std::atomic<uint64_t> done{0};
    const int st = set_dynamic_lds(reinterpret_cast<const void*>(&narrow_kernel<T, D>), (int)narrow_lds(D), done);
    if (st != kOk) return st;
    narrow_kernel<T, D><<<step.narrow, kThreads, narrow_lds(D), stream>>>(a);
  }
  if (step.wide > 0) {
    static std::atomic<uint64_t> done{0};
    constexpr int kR = D == 256 ? 1 : 2, kW = 8 / kR, kWgs = D == 64 ? 2 : 1;
    const auto kernel = &wide_kernel<T, D, kR, kW, kWgs>;
    const int st = set_dynamic_lds(reinterpret_cast<const void*>(kernel), wide_lds<D>(), done);
    if (st != kOk) return st;
    kernel<<<step.wide, 64 * kW, wide_lds<D>(), stream>>>(a);
  }
  if (step.joins > 0) join_kernel<T, D><<<dim3(step.joins, kTileRows, D / 64), 256, 0, stream>>>(a);
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
  return c->block_size % 16 == 0 ? kOk : kErrUnsupportedGeometry;
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
    step->window = std::min(window, kMostKeys);
    step->table_cols = pages;
    step->narrow = (int32_t)plan.narrow.size();
    step->wide = (int32_t)plan.wide.size();
    step->joins = (int32_t)plan.joins.size();
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
  if (step->narrow < 0 || step->wide < 0 || step->joins < 0) return kErrInvalidArgument;
  if (step->narrow + step->wide == 0) return kOk;
  if (items == nullptr || block_table == nullptr || query->data == nullptr || out->data == nullptr ||
      block_table_stride < step->table_cols)
    return kErrInvalidArgument;
  if ((int64_t)workspace_size < step->workspace_size || (step->workspace_size > 0 && workspace == nullptr))
    return kErrWorkspaceTooSmall;
  if (((uintptr_t)query->data | (uintptr_t)out->data | (uintptr_t)workspace | (uintptr_t)items) % 16 ||
      (query->token_stride | query->head_stride | out->token_stride | out->head_stride) % 8)
    return kErrUnsupportedGeometry;
  ChunkArgs a{};
  a.q = static_cast<const uint8_t*>(query->data);
  a.out = static_cast<uint8_t*>(out->data);
  a.q_token = 2 * query->token_stride;
  a.q_head = 2 * query->head_stride;
  a.out_token = 2 * out->token_stride;
  a.out_head = 2 * out->head_stride;
  a.k = static_cast<const uint8_t*>(cache->k);
  a.v = static_cast<const uint8_t*>(cache->v);
  a.k_page = cache->k_stride_page;
  a.v_page = cache->v_stride_page;
  a.num_pages = cache->num_pages;
  a.k_token = (int32_t)cache->k_stride_token;
  a.v_token = (int32_t)cache->v_stride_token;
  a.k_head = (int32_t)cache->k_stride_head;
  a.v_head = (int32_t)cache->v_stride_head;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.pieces = static_cast<const Piece*>(items);
  a.wide0 = step->narrow;
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
