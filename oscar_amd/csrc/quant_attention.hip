// Causal attention of a step's new tokens over the 8-bit paged cache
// (oscar_quant_attention).
//
// Its keys are k = c_k 2^a and its values v = c_v 2^b, c codes and a, b one for each
// token and head.  With few rows, memory bounds the attention, so codes are what goes to
// LDS, half of what 16-bit pages take, and they become operands on the way to the matrix
// unit: a lane's K operand is of one key, whose 2^a the conversion takes along, exactly.
// V^T's operand is of eight keys a lane, so 2^b goes into the weights instead: with x the
// scores in powers of two,
//   o = sum_t 2^(x_t + b_t - m) c_v,t / sum_t 2^(x_t - m),
// m the running maximum of x_t + b_t, so that the weights that are rounded for the
// product are the ones whose size counts, whatever the powers.  The sum below is of fp32
// weights.  Numerators and sums of pieces relate by 2^m as those over 16-bit pages do,
// and the same launch joins them.
//
// Requests of more rows are bounded by the matrix unit, which would wait for the
// conversions that each of a tile's four waves makes for itself.  Their keys are
// converted once, into 16-bit pages in the workspace (read_pages), and computed there by
// the wide pieces of the plain cache.
#include "chunk_pieces.h"
#include "chunk_plan.h"
#include "quant_cache.h"
#include "quant_values.h"

namespace oscar {
namespace {

// Keys [16 group0, 16 (group0 + groups)) of a block table row, on workspace pages of 16
// keys from page0 on.
struct Source {
  int32_t table_row, group0, groups, page0;
};
static_assert(sizeof(Source) == 16, "item size");

struct QuantArgs {
  const uint8_t* k;        // codes
  const uint8_t* v;
  const uint8_t* exponents;
  int64_t num_pages;
  uint32_t k_page, v_page;                           // bytes
  int32_t k_token, v_token, k_head, v_head;          // bytes
  const int32_t* table;
  int64_t table_stride;
  int32_t block_size, num_heads;
  FastDiv block_div;
};
// `wide` is over the workspace's pages; narrow pieces take rows, outputs and partials of
// it, and their keys from `codes`.
struct QuantChunkArgs {
  ChunkArgs wide;
  QuantArgs codes;
};

// ---------------------------------------------------------------- 32 rows
// A tile's codes lie in LDS as rows of D bytes, chunk c (16 bytes) of key r at place c ^
// swizzle(r): so that K's reads find 16 keys' chunks on different banks, and V's (8 keys
// x 32 bytes a half wave, in pairs of chunks) theirs.
template <int D>
__device__ __forceinline__ int k_code_swizzle(int key) {
  return D == 256 ? key & 15 : D == 128 ? (key >> 1) & 7 : (key >> 2) & 3;
}
template <int D>
__device__ __forceinline__ int v_code_swizzle(int key) {
  const int eight = (key >> 3) & 1;
  return 2 * (D == 256 ? (key & 3) | eight << 2 : D == 128 ? ((key >> 1) & 1) | eight << 1 : eight);
}

// Where a lane's 16 bytes of the first load of a run of keys lie, as lane_place.
template <int D, bool kV>
__device__ __forceinline__ LanePlace code_place(const QuantArgs& a, int lane) {
  constexpr int kLaneRow = D / 16;
  const int key = lane / kLaneRow, place = lane % kLaneRow;
  return LanePlace{key * (kV ? a.v_token : a.k_token),
                   16 * (place ^ (kV ? v_code_swizzle<D>(key) : k_code_swizzle<D>(key)))};
}

// 16 keys' codes from `key` on, as load_keys.
template <int D, bool kV>
__device__ __forceinline__ void load_codes(const QuantArgs& a, const Piece& p, int key, int key_in_tile, int page,
                                           int in_page, uint8_t* lds, const LanePlace& at) {
  constexpr int kStep = 1024 / D;           // keys of a load
  const int stride = kV ? a.v_token : a.k_token;
  const int live = page < 0 ? 0 : min(16, p.key1 - key);
  const uint8_t* base = (kV ? a.v : a.k) + (int64_t)p.kv_head * (kV ? a.v_head : a.k_head) +
                        (uint64_t)(uint32_t)max(page, 0) * (kV ? a.v_page : a.k_page) + (uint32_t)(in_page * stride);
  const uint32_t records = live > 0 ? (uint32_t)((live - 1) * stride + D) : 0u;
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, records, 0x00020000);
#pragma unroll
  for (int n = 0; n < 16 / kStep; ++n) {
    const int first = key_in_tile + n * kStep;
    const int turn = 16 * (kV ? v_code_swizzle<D>(first) : k_code_swizzle<D>(first));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(lds + first * D), 16,
                                             at.row + n * kStep * stride + (at.chunk ^ turn), 0, 0, kOnce);
  }
}

// The rows of a piece, the features of query operands in the order of K's codes: a
// chunk's 16 are two steps' 8.
template <typename T, int D>
__device__ __forceinline__ void load_code_rows(const ChunkArgs& a, const Piece& p, int lane, RowState<T, D>& s) {
  const int end = p.row0 + p.rows - 1;
  const int row = min(p.row0 + (lane & 31), end);     // rows past the last repeat it and are not stored
  const int tok = (int)fast_div((uint32_t)row, a.group_div);
  const int head = row - tok * a.group + p.kv_head * a.group;
  const uint8_t* src = a.q + (int64_t)(p.token0 + tok) * a.q_token + (int64_t)head * a.q_head + 32 * (lane >> 5);
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    s.q[i] = *reinterpret_cast<const typename Num<T>::V8*>(src + 64 * (i / 2) + 16 * (i % 2));
#pragma unroll
  for (int i = 0; i < D / 32; ++i) s.acc[i] = floatx16{};
  s.m = kNone;
  s.l = 0.f;
  s.pos = p.pos0 + tok;
  s.first = p.pos0 + (int)fast_div((uint32_t)p.row0, a.group_div);
  s.last = p.pos0 + (int)fast_div((uint32_t)min(p.row0 + kTileRows - 1, end), a.group_div);
}

template <typename T>
__device__ __forceinline__ typename Num<T>::V8 operand_of(u32x2 codes, float scale) {
  return __builtin_bit_cast(typename Num<T>::V8, values8<T>(codes, scale));
}

// V^T's codes of feature block b (in `place`, xor-ed with 32 b): eight keys of one feature.
__device__ __forceinline__ u32x2 v_codes_at(const uint8_t* vt, int place) {
  typedef int intx2 __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) intx2 lds_int2;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2*)(vt + place)));
}
template <int D>
__device__ __forceinline__ int v_code_read(int lane) {
  const int row = (lane & 15) >> 1, key = 4 * (lane >> 5) + (row & 3) + 2 * (row & 4);
  return key * D + ((16 * ((lane >> 4) & 1)) ^ (16 * v_code_swizzle<D>(key))) + 8 * (lane & 1);
}

// As take_out_special: codes of NaN (there are no infinities) become zeros.
template <int kBytes>
__device__ __forceinline__ bool take_out_nan(uint8_t* vt, int lane) {
  u32x4* const at = reinterpret_cast<u32x4*>(vt) + lane;
  uint32_t found = 0;
#pragma unroll
  for (int i = 0; i < kBytes / 1024; ++i) {
    const u32x4 x = (at[64 * i] & 0x7F7F7F7Fu) + 0x01010101u;
    found |= x[0] | x[1] | x[2] | x[3];
  }
  if (__builtin_expect(__ballot((found & 0x80808080u) != 0u) == 0ull, 1)) return false;
#pragma unroll 1
  for (int i = 0; i < kBytes / 1024; ++i) {
    const u32x4 x = at[64 * i], nan = (((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
    at[64 * i] = x & ~(nan * 0xFFu);
  }
  return true;
}
// NaN among a tile's values, for the rows that see them; what is whole and mapped had
// them in the product.
template <typename T, int D>
__device__ __forceinline__ void add_nan(const ChunkArgs& a, const QuantArgs& c, const Piece& p, int key0, bool whole,
                                        int lane, RowState<T, D>& s) {
  auto page_of = [&](int key) {
    const int page = c.table[(int64_t)p.table_row * c.table_stride + fast_div((uint32_t)key, c.block_div)];
    return page >= 0 && page < c.num_pages ? page : -1;
  };
  const int end = min(key0 + kTileKeys, p.key1);
  if (whole && page_of(key0) >= 0 && page_of(end - 1) >= 0) return;
  for (int key = key0; key < end; ++key) {
    const int page = page_of(key);
    if (page < 0) continue;
    const uint8_t* row = c.v + (int64_t)p.kv_head * c.v_head + (uint64_t)(uint32_t)page * c.v_page +
                         (uint64_t)fast_mod((uint32_t)key, c.block_div) * (uint32_t)c.v_token + 4 * (lane >> 5);
    const bool seen = key <= s.pos && (a.window == 0 || key > s.pos - a.window);
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(row + 32 * b + 8 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (seen && ((x >> (8 * i)) & 0x7Fu) == 0x7Fu) s.acc[b][4 * j + i] = __builtin_nanf("");
        keep_order();                       // (few registers: this is rarely run)
      }
  }
}

// One row tile, its keys shared out to four waves: narrow_piece's walk over codes.  The
// powers of a tile's keys are one load of two bytes a lane, on its way with the tile's K;
// V's go through LDS to the lanes that hold the keys' scores.
constexpr int code_lds(int d) { return kWaves * 2 * kTileKeys * d + kWaves * 2 * kTileRows * 4; }

template <typename T, int D>
__device__ __forceinline__ void code_piece(const QuantChunkArgs& all, const Piece p, uint8_t* smem) {
  typedef typename Num<T>::V8 V8;
  const ChunkArgs& a = all.wide;
  const QuantArgs& c = all.codes;
  constexpr int kTileBytes = kTileKeys * D, kLoads = kTileBytes / 1024, kBlocks = D / 32;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles = (p.key1 - p.key0 + kTileKeys - 1) / kTileKeys;
  const int first = p.key0 / kTileKeys + tiles * wave / kWaves;
  const int last = p.key0 / kTileKeys + tiles * (wave + 1) / kWaves;

  auto load_group_pages = [&](int base) {   // of 64 groups of 16 keys, one a lane; -1: unmapped
    const int key = 16 * (base + lane);
    int page = -1;
    if (key < p.key1) {
      page = c.table[(int64_t)p.table_row * c.table_stride + fast_div((uint32_t)key, c.block_div)];
      page = page >= 0 && page < c.num_pages ? page : -1;
    }
    return page;
  };
  int page_base = 2 * first;
  int pages = load_group_pages(page_base);
  RowState<T, D> s;
  load_code_rows<T, D>(a, p, lane, s);
  const int whole_from = a.window == 0 ? 0 : s.last - a.window + 1, whole_to = s.first - kTileKeys + 1;
  auto whole = [&](int key0) { return key0 >= whole_from && key0 <= whole_to; };
  bool special = false;                     // a tile that is not whole held values that are NaN

  const LanePlace k_place = code_place<D, false>(c, lane), v_place = code_place<D, true>(c, lane);
  auto page_of = [&](int t, int h) { return __builtin_amdgcn_readlane(pages, 2 * t + h - page_base); };
  auto in_page = [&](int t, int h) {
    return __builtin_amdgcn_readfirstlane((int)fast_mod((uint32_t)(kTileKeys * t + 16 * h), c.block_div));
  };
  auto load_tile = [&](int t, auto v_tag, uint8_t* lds) {
    constexpr bool kV = decltype(v_tag)::value;
    const LanePlace& place = kV ? v_place : k_place;
    const LanePlace at{opaque(place.row), opaque(place.chunk)};      // (its sums stay out of registers)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      load_codes<D, kV>(c, p, t * kTileKeys + 16 * h, 16 * h, page_of(t, h), in_page(t, h), lds, at);
  };
  // The powers of key lane % 32: K's in the low byte, V's above.
  // (Their places as scalars: as a choice of the lane the pages would be the lane's for the
  // loads to LDS as well, which then loop over descriptors.)
  auto load_powers = [&](int t) {
    int64_t at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int page = max(page_of(t, h), 0), first = in_page(t, h);
      asm volatile("" : "+s"(page), "+s"(first));
      at[h] = 2 * (((int64_t)page * c.num_heads + p.kv_head) * c.block_size + first);
    }
    return (uint32_t)*reinterpret_cast<const uint16_t*>(c.exponents + ((lane & 16) != 0 ? at[1] : at[0]) + 2 * (lane & 15));
  };
  const int key = lane & 31;
  const int k_addr = key * D + 16 * ((lane >> 5) ^ k_code_swizzle<D>(key)), v_addr = v_code_read<D>(lane);
  float* const v_powers = reinterpret_cast<float*>(smem + kWaves * 2 * kTileBytes) + wave * kTileKeys;
  uint32_t powers = 0;

  // (The two places as parameters that do not alias, as in narrow_piece.)
  auto tile = [&](int t, uint8_t* __restrict__ kt, uint8_t* __restrict__ vt) __attribute__((always_inline)) {
    const uint32_t unmapped = (page_of(t, 0) < 0 ? 1u : 0u) | (page_of(t, 1) < 0 ? 2u : 0u);
    const bool more = t + 1 < last;
    if (more && 2 * (t + 1) - page_base >= 64) {
      page_base = 2 * (t + 1);
      pages = load_group_pages(page_base);
    }
    // Loads end in order: V's kLoads came after K's (and the powers beside them, wherever
    // they stand among these), and below the next tile's K's after V's.
    wait_vmcnt<kLoads>();                   // K is there, V on its way
    asm volatile("" ::: "memory");
    const float k_scale = scale_of(powers & 0xFFu);
    if (lane < 32) v_powers[lane] = (float)((int)(powers >> 8) - 127);
    floatx16 x{};
    // (two reads ahead, in this order: left to it, the compiler asks for all at once and
    // spills registers at D = 256)
    u32x4 codes[2];
    auto k_codes = [&](int i) { return *reinterpret_cast<const u32x4*>(kt + (opaque(k_addr) ^ (32 * i))); };
    codes[0] = k_codes(0);
    codes[1] = k_codes(1);
    keep_order();
    each<D / 32>([&](auto step) {
      constexpr int i = decltype(step)::value;
      const u32x4 now = codes[i % 2];
      if constexpr (i + 2 < D / 32) codes[i % 2] = k_codes(i + 2);
      x = Num<T>::mfma(operand_of<T>(u32x2{now[0], now[1]}, k_scale), s.q[2 * i], x);
      x = Num<T>::mfma(operand_of<T>(u32x2{now[2], now[3]}, k_scale), s.q[2 * i + 1], x);
      keep_order();
    });
    asm volatile("" ::: "memory");
    if (more) {
      powers = load_powers(t + 1);
      load_tile(t + 1, std::false_type{}, kt);
    }

    const int key0 = t * kTileKeys;
    const bool masked = !whole(key0) || unmapped != 0u;
    if (masked) mask_scores<16>(a, x, key0, unmapped, lane, s.pos);
    // (V's powers are read twice: registers)
    auto v_power = [&](int j) { return *reinterpret_cast<const floatx4*>(v_powers + 8 * j + 4 * (lane >> 5)); };
    float top = kNone;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const floatx4 b = v_power(j);
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fmaf(x[4 * j + i], a.scale_log2, b[i]));
    }
    top = max_halves(top);
    const bool raise = top > s.m + (kLazy + Num<T>::kLift);
    if (__ballot(raise)) {
      const float m = raise ? top - Num<T>::kLift : s.m, f = __builtin_amdgcn_exp2f(s.m - m);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) s.acc[b] *= f;
      s.l *= f;
      s.m = m;
    }
    keep_order();
    V8 w[2];
    float l = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const floatx4 b = v_power(2 * h + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = __builtin_fmaf(x[8 * h + 4 * j + i], a.scale_log2, -s.m);
          l += __builtin_amdgcn_exp2f(y);
          f[4 * j + i] = __builtin_amdgcn_exp2f(y + b[i]);
        }
      }
      w[h] = Num<T>::round8(f);
    }
    s.l += l;

    if (more) wait_vmcnt<kLoads>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    if (masked) special = take_out_nan<kTileBytes>(vt, lane) || special;
    keep_order();
    each<2 * kBlocks>([&](auto step) {
      constexpr int h = decltype(step)::value / kBlocks, b = decltype(step)::value % kBlocks;
      s.acc[b] = Num<T>::mfma(operand_of<T>(v_codes_at(vt + h * 16 * D, opaque(v_addr) ^ (32 * b)), 1.f), w[h], s.acc[b]);
      if constexpr (b % 4 == 3 || b == kBlocks - 1) keep_order();
    });
    asm volatile("" ::: "memory");
    if (more) load_tile(t + 1, std::true_type{}, vt);
  };
  uint8_t* const kt = smem + wave * 2 * kTileBytes;
  if (first < last) {
    powers = load_powers(first);
    load_tile(first, std::false_type{}, kt);
    __builtin_amdgcn_sched_barrier(0);      // (the waits count K's loads before V's)
    load_tile(first, std::true_type{}, kt + kTileBytes);
  }
  for (int t = first; t < last; ++t) tile(t, kt, kt + kTileBytes);
  if (__builtin_expect(special, 0))
    for (int t = first; t < last; ++t) add_nan<T, D>(a, c, p, t * kTileKeys, whole(t * kTileKeys), lane, s);
  combine_waves<T, D, 2>(a, p, s, smem, tid, lane, wave);
}

// ---------------------------------------------------------------- kernels
constexpr int code_wgs(int d) { return d == 256 ? 2 : d == 128 ? 3 : 4; }      // workgroups a CU
template <typename T, int D>
__global__ __launch_bounds__(kThreads, code_wgs(D)) void code_kernel(QuantChunkArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[code_lds(D)];
  code_piece<T, D>(a, a.wide.pieces[blockIdx.x], smem);
}
// A step with wide pieces, the narrow ones first where they are few, as mixed_kernel.
constexpr int kFewNarrow = kCus;
template <typename T, int D>
__global__ __launch_bounds__(kThreads, kWideWgs) void quant_kernel(QuantChunkArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[std::max(code_lds(D), wide_lds(D))];
  const int total = a.wide.narrow + a.wide.wide, lead = a.wide.narrow <= kFewNarrow ? 0 : a.wide.narrow;
  const int at = (int)blockIdx.x + lead, i = at < total ? at : at - total;
  if (i >= a.wide.narrow) wide_piece<T, D>(a.wide, a.wide.pieces[i], smem);
  else code_piece<T, D>(a, a.wide.pieces[i], smem);
}

// The sources' keys as 16-bit pages of 16 keys [K | V][key][head][D], a workgroup each,
// and the pages' block table.  A thread takes 8 codes at a time, four times at once.
struct PagesArgs {
  QuantArgs codes;
  const Source* sources;
  int32_t num_sources, d;
  int32_t* table;
  uint8_t* pages;
  FastDiv by_key, by_head; // items of a key, of a head
};
template <typename T>
__global__ __launch_bounds__(256) void pages_kernel(PagesArgs a) {
  const QuantArgs& c = a.codes;
  const int at = (int)blockIdx.x;
  int low = 0, high = a.num_sources - 1;    // the last source whose page0 <= at
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (a.sources[mid].page0 <= at) low = mid;
    else high = mid - 1;
  }
  const Source src = a.sources[low];
  const int key0 = 16 * (src.group0 + at - src.page0);
  const int page = c.table[(int64_t)src.table_row * c.table_stride + fast_div((uint32_t)key0, c.block_div)];
  const bool mapped = page >= 0 && page < c.num_pages;
  if (threadIdx.x == 0) a.table[at] = mapped ? at : -1;
  if (!mapped) return;
  const int in_page = (int)fast_mod((uint32_t)key0, c.block_div);
  const uint8_t* const from[2] = {c.k + (uint64_t)(uint32_t)page * c.k_page, c.v + (uint64_t)(uint32_t)page * c.v_page};
  const uint8_t* const powers = c.exponents + 2 * ((int64_t)page * c.num_heads * c.block_size + in_page);
  const int per_key = (int)a.by_key.d, side = 16 * per_key;      // items of K
  uint8_t* const to = a.pages + (int64_t)at * 2 * side * 16;
  for (int first = (int)threadIdx.x; first < 2 * side; first += 4 * 256) {
    u32x2 codes[4];
    uint32_t power[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int item = min(first + 256 * n, 2 * side - 1);
      const int v = item >= side ? 1 : 0, rest = item - v * side;
      const int key = (int)fast_div((uint32_t)rest, a.by_key), in_key = rest - key * per_key;
      const int head = (int)fast_div((uint32_t)in_key, a.by_head), piece = in_key - head * (int)a.by_head.d;
      codes[n] = *reinterpret_cast<const u32x2*>(from[v] + (int64_t)(in_page + key) * (v ? c.v_token : c.k_token) +
                                                 (int64_t)head * (v ? c.v_head : c.k_head) + 8 * piece);
      power[n] = powers[2 * ((int64_t)head * c.block_size + key) + v];
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int item = first + 256 * n;
      if (item < 2 * side) store_values<T, false>(to + (int64_t)item * 16, codes[n], scale_of(power[n]));
    }
  }
}

// ---------------------------------------------------------------- host
inline PlanRule quant_rule(int32_t head_size) {
  return PlanRule{head_size, kTileRows, {kCus * code_wgs(head_size), kCus * code_wgs(head_size)}, 1.};
}

// The wide pieces' keys, request by request, and the pieces' table rows in the pages'.
void make_sources(Plan& plan, std::vector<Source>& sources, int64_t& pages) {
  std::vector<std::pair<int32_t, size_t>> order;       // table row, piece
  for (size_t i = 0; i < plan.wide.size(); ++i) order.emplace_back(plan.wide[i].table_row, i);
  std::sort(order.begin(), order.end());
  pages = 0;
  for (size_t i = 0; i < order.size();) {
    const int32_t row = order[i].first;
    int32_t from = kMostKeys, to = 0;
    size_t end = i;
    for (; end < order.size() && order[end].first == row; ++end) {
      const Piece& p = plan.wide[order[end].second];
      from = std::min(from, p.key0 / 16);
      to = std::max(to, (p.key1 + 15) / 16);
    }
    if (pages + to - from > INT32_MAX) throw 0;
    for (; i < end; ++i) plan.wide[order[i].second].table_row = (int32_t)pages - from;
    sources.push_back(Source{row, from, to - from, (int32_t)pages});
    pages += to - from;
  }
}

int check_quant_geometry(const oscar_quant_cache* c) {
  const int status = check_quant_cache(c);
  if (status != kOk) return status;
  if (c->head_size != 64 && c->head_size != 128 && c->head_size != 256) return kErrUnsupportedHeadDim;
  const bool near = c->k_stride_page <= UINT32_MAX && c->v_stride_page <= UINT32_MAX;
  return c->block_size % 16 == 0 && near ? kOk : kErrUnsupportedGeometry;
}

int64_t page_bytes(const oscar_chunk_step& s) { return 2ll * 16 * s.num_kv_heads * s.head_size * 2; }
int64_t table_bytes(const oscar_quant_step& s) { return ((int64_t)s.pages * 4 + 255) / 256 * 256; }

template <typename T, int D>
int launch(const QuantChunkArgs& a, const PagesArgs& pages, const oscar_quant_step& step, hipStream_t stream) {
  static_assert(code_wgs(D) * code_lds(D) <= 160 * 1024 && kWideWgs * std::max(code_lds(D), wide_lds(D)) <= 160 * 1024,
                "the workgroups of a CU must fit its 160 KiB of LDS");
  if (step.pages > 0) pages_kernel<T><<<step.pages, 256, 0, stream>>>(pages);
  const uint32_t pieces = (uint32_t)(step.chunk.narrow + step.chunk.wide);
  if (step.chunk.wide == 0) code_kernel<T, D><<<pieces, kThreads, 0, stream>>>(a);
  else quant_kernel<T, D><<<pieces, kThreads, 0, stream>>>(a);
  return launch_joins<T, D>(a.wide, step.chunk, stream);
}
template <typename T>
int launch_sized(int d, const QuantChunkArgs& a, const PagesArgs& pages, const oscar_quant_step& step,
                 hipStream_t stream) {
  if (d == 64) return launch<T, 64>(a, pages, step, stream);
  if (d == 128) return launch<T, 128>(a, pages, step, stream);
  return launch<T, 256>(a, pages, step, stream);
}

}  // namespace
}  // namespace oscar

extern "C" int oscar_quant_plan(const int32_t* query_start_loc, const int32_t* seq_lens, int32_t num_requests,
                                int32_t num_heads, int32_t window, const oscar_prefix* prefixes, int32_t num_prefixes,
                                const oscar_quant_cache* cache, void* items, size_t items_size,
                                oscar_quant_step* step) {
  using namespace oscar;
  int status = check_quant_geometry(cache);
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
    make_plan(query_start_loc, seq_lens, num_requests, group, cache->num_kv_heads, quant_rule(cache->head_size), window,
              shared, plan);
    std::vector<Source> sources;
    int64_t read = 0;
    make_sources(plan, sources, read);
    oscar_chunk_step& s = step->chunk;
    s.num_requests = num_requests;
    s.num_tokens = num_requests > 0 ? query_start_loc[num_requests] : 0;
    s.num_heads = num_heads;
    s.num_kv_heads = cache->num_kv_heads;
    s.head_size = cache->head_size;
    s.block_size = cache->block_size;
    s.window = std::min(window, kMostKeys);
    s.table_cols = pages;
    status = pack_plan(plan, cache->head_size, items, items_size, &s);
    const int64_t packed = s.items_size;
    step->sources = (int32_t)sources.size();
    step->pages = (int32_t)read;
    step->partials_size = (s.workspace_size + 255) / 256 * 256;
    s.items_size += (int64_t)(sources.size() * sizeof(Source));
    s.workspace_size = read == 0 ? s.workspace_size : step->partials_size + table_bytes(*step) + read * page_bytes(s);
    if (status != kOk || items == nullptr) return status;
    if ((int64_t)items_size < s.items_size) return kErrWorkspaceTooSmall;
    if (!sources.empty())
      std::memcpy(static_cast<uint8_t*>(items) + packed, sources.data(), sources.size() * sizeof(Source));
  } catch (...) {
    return kErrInvalidArgument;
  }
  return kOk;
}

extern "C" int oscar_quant_attention(const oscar_quant_step* step, const void* items, const int32_t* block_table,
                                     int64_t block_table_stride, const oscar_quant_cache* cache,
                                     const oscar_heads* query, const oscar_heads* out, float scale, void* workspace,
                                     size_t workspace_size, oscar_stream_t stream) {
  using namespace oscar;
  const int status = check_quant_geometry(cache);
  if (status != kOk) return status;
  if (step == nullptr || query == nullptr || out == nullptr || !(scale > 0.f) || !(scale <= 3.0e38f))
    return kErrInvalidArgument;
  const oscar_chunk_step& s = step->chunk;
  if (query->num_heads != s.num_heads || out->num_heads != s.num_heads || s.num_heads < 1 ||
      s.num_heads % cache->num_kv_heads || s.num_kv_heads != cache->num_kv_heads || s.head_size != cache->head_size ||
      s.block_size != cache->block_size)
    return kErrInvalidArgument;
  if (s.narrow < 0 || s.wide < 0 || s.few_joins < 0 || s.joins < s.few_joins || s.parts < 0 || step->sources < 0 ||
      step->pages < 0 || (s.wide > 0) != (step->sources > 0) || (s.wide > 0) != (step->pages > 0) ||
      step->partials_size < 0)
    return kErrInvalidArgument;
  if (s.narrow + s.wide == 0) return kOk;
  QuantChunkArgs a{};
  int64_t need = s.workspace_size;
  if (step->pages > 0)                      // (what the launches write, whatever the step says)
    need = std::max(need, step->partials_size + table_bytes(*step) + step->pages * page_bytes(s));
  const int bad = step_args(&s, items, block_table, block_table_stride, query, out, scale, workspace, workspace_size,
                            need, a.wide);
  if (bad != kOk) return bad;
  QuantArgs& c = a.codes;
  c.k = static_cast<const uint8_t*>(cache->k);
  c.v = static_cast<const uint8_t*>(cache->v);
  c.exponents = cache->exponents;
  c.num_pages = cache->num_pages;
  c.k_page = (uint32_t)cache->k_stride_page;
  c.v_page = (uint32_t)cache->v_stride_page;
  c.k_token = (int32_t)cache->k_stride_token;
  c.v_token = (int32_t)cache->v_stride_token;
  c.k_head = (int32_t)cache->k_stride_head;
  c.v_head = (int32_t)cache->v_stride_head;
  c.table = block_table;
  c.table_stride = block_table_stride;
  c.block_size = cache->block_size;
  c.num_heads = cache->num_kv_heads;
  c.block_div = make_fast_div((uint32_t)cache->block_size);
  PagesArgs pages{};
  if (step->pages > 0) {
    uint8_t* const at = static_cast<uint8_t*>(workspace) + step->partials_size;
    pages.codes = c;
    pages.sources = reinterpret_cast<const Source*>(a.wide.parts + s.parts);
    pages.num_sources = step->sources;
    pages.d = cache->head_size;
    pages.table = reinterpret_cast<int32_t*>(at);
    pages.pages = at + table_bytes(*step);
    pages.by_key = make_fast_div((uint32_t)(cache->num_kv_heads * (cache->head_size / 8)));
    pages.by_head = make_fast_div((uint32_t)(cache->head_size / 8));
    // the wide pieces' cache
    ChunkArgs& w = a.wide;
    const int32_t head = 2 * cache->head_size, token = head * cache->num_kv_heads;
    w.k = pages.pages;
    w.v = pages.pages + 16 * (int64_t)token;
    w.k_page = w.v_page = (uint32_t)(2 * 16 * token);
    w.k_token = w.v_token = token;
    w.k_head = w.v_head = head;
    w.num_pages = step->pages;
    w.table = pages.table;
    w.table_stride = 1;                     // (pieces name their source's first page)
    w.block_size = 16;
    w.block_div = make_fast_div(16);
  }
  return cache->dtype == OSCAR_BF16 ? launch_sized<__bf16>(cache->head_size, a, pages, *step, stream)
                                    : launch_sized<_Float16>(cache->head_size, a, pages, *step, stream);
}
