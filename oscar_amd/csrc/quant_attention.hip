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
// weights, not of the rounded ones as over 16-bit pages: those go with 2^b, and keys whose
// values are far below the heaviest's, rows of zeros too, would be missing from it.
// Numerators and sums of pieces relate by 2^m as those over 16-bit pages do, and the same
// launch joins them.
//
// Requests of more rows are bounded by the matrix unit, which would wait for the
// conversions that each of a tile's four waves makes for itself.  Their keys are
// converted once, into 16-bit pages in the workspace (read_pages), and computed there by
// the wide pieces of the plain cache.
#include "chunk_pieces.h"
#include "chunk_plan.h"
#include "quant_cache.h"
#include "quant_values.h"

#include <utility>

namespace oscar {
namespace {

// Keys [16 group0, 16 (group0 + groups)) of a block table row, on workspace pages of 16
// keys from page0 on.
struct Source {
  int32_t table_row, group0, groups, page0;
};
static_assert(sizeof(Source) == 16, "item size");
constexpr int64_t kLastCache = 256ll << 20;      // bytes

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
template <int D, bool kV, int kPolicy>
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
                                             at.row + n * kStep * stride + (at.chunk ^ turn), 0, 0, kPolicy);
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
// NaN among the values of a tile of kKeys, for the rows that see them.  A tile that is whole
// and has all its groups of 16 keys, mapped ones below the piece's last, had them in the
// product; of any other they were taken out, of the groups that are there as well.
template <typename T, int D, int kKeys>
__device__ __forceinline__ void add_nan(const ChunkArgs& a, const QuantArgs& c, const Piece& p, int key0, bool whole,
                                        int lane, RowState<T, D>& s) {
  auto page_of = [&](int key) {
    const int page = c.table[table_row_of(p, key) * c.table_stride + fast_div((uint32_t)key, c.block_div)];
    return page >= 0 && page < c.num_pages ? page : -1;
  };
  bool there = whole;
  for (int key = key0; there && key < key0 + kKeys; key += 16) there = key < p.key1 && page_of(key) >= 0;
  if (there) return;
  for (int key = key0; key < min(key0 + kKeys, p.key1); ++key) {
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

// One row tile, its keys shared out to four waves: narrow_piece's walk over codes, 8 KB of
// K's and 8 of V's at a time whatever D is (32, 64 or 128 keys), so that as many bytes are
// on their way.  The powers of a tile's keys are loads of two bytes a lane, with the tile's
// K; V's go through LDS to the lanes that hold the keys' scores, as numbers and as powers.
// A tile is weighed by the maximum as it stands, and only where a weight is too large
// is the maximum raised and the tile weighed again.
// Memory bounds it: 32 users' 4 tokens of 6 heads over 2K to 16K keys of 256, 146 MB, 31.3
// us (4.7 TB/s; 10 to 15 % less without the products: the rest is the start, the first
// tile's round trips and the waves' joining), 32 users' token over 8 heads of 128, 578 MB, 118
// (5.0 TB/s); at D = 64, 32 users' 4 tokens of 16 heads on 4, 147 MB, 43 with the join (3.4
// TB/s; 41 where a head's rows lie together).
constexpr int code_keys(int d) { return 8192 / d; }
constexpr int kCodeWgs = 2;                // workgroups a CU
constexpr int code_lds(int d) { return kWaves * (2 * 8192 + std::max(2 * code_keys(d) * 4, 2 * kTileRows * 4)); }

template <typename T, int D, int kPolicy>
__device__ __forceinline__ void code_piece(const QuantChunkArgs& all, const Piece p, uint8_t* smem) {
  typedef typename Num<T>::V8 V8;
  const ChunkArgs& a = all.wide;
  const QuantArgs& c = all.codes;
  constexpr int kKeys = code_keys(D), kSubs = kKeys / 32, kGroups = kKeys / 16;
  constexpr int kTileBytes = kKeys * D, kLoads = kTileBytes / 1024, kBlocks = D / 32;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (tiles of kKeys from key0 on, which is a multiple of 32)
  const int tiles = (p.key1 - p.key0 + kKeys - 1) / kKeys;
  const int first = tiles * wave / kWaves, last = tiles * (wave + 1) / kWaves;
  const int group0 = p.key0 / 16;

  auto load_group_pages = [&](int base) {   // of 64 groups of 16 keys, one a lane; -1: unmapped
    const int key = 16 * (group0 + base + lane);
    int page = -1;
    if (key < p.key1) {
      page = c.table[table_row_of(p, key) * c.table_stride + fast_div((uint32_t)key, c.block_div)];
      page = page >= 0 && page < c.num_pages ? page : -1;
    }
    return page;
  };
  int page_base = kGroups * first;
  int pages = load_group_pages(page_base);
  RowState<T, D> s;
  load_code_rows<T, D>(a, p, lane, s);
  const int whole_from = a.window == 0 ? 0 : s.last - a.window + 1, whole_to = s.first - kKeys + 1;
  auto whole = [&](int key0) { return key0 >= whole_from && key0 <= whole_to; };
  bool special = false;                     // a tile that is not whole held values that are NaN

  auto page_of = [&](int t, int h) { return __builtin_amdgcn_readlane(pages, kGroups * t + h - page_base); };
  auto in_page = [&](int t, int h) {
    return __builtin_amdgcn_readfirstlane((int)fast_mod((uint32_t)(p.key0 + kKeys * t + 16 * h), c.block_div));
  };
  auto load_tile = [&](int t, auto v_tag, uint8_t* lds) {
    constexpr bool kV = decltype(v_tag)::value;
    const LanePlace at = code_place<D, kV>(c, opaque(lane));       // (found anew: registers)
#pragma unroll
    for (int h = 0; h < kGroups; ++h)
      load_codes<D, kV, kPolicy>(c, p, p.key0 + t * kKeys + 16 * h, 16 * h, page_of(t, h), in_page(t, h), lds, at);
  };
  // The powers of keys lane % 32 of the subtiles: K's in the low byte, V's above, which is
  // taken for the type's least where it is outside its range (zeros that no write has left:
  // below it a weight over 2^-127 would pass fp32, above it the maximum would be theirs and
  // every other key's weight nothing beside it).  (Their
  // places as scalars: as a choice of the lane the pages would be the lane's for the
  // loads to LDS as well, which then loop over descriptors.)
  uint32_t powers[kSubs];
  auto load_powers = [&](int t) {
#pragma unroll
    for (int u = 0; u < kSubs; ++u) {
      int64_t at[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int page = max(page_of(t, 2 * u + h), 0), from = in_page(t, 2 * u + h);
        asm volatile("" : "+s"(page), "+s"(from));
        at[h] = 2 * (((int64_t)page * c.num_heads + p.kv_head) * c.block_size + from);
      }
      const int at_lane = opaque(lane);
      const int64_t row = (at_lane & 16) != 0 ? at[1] : at[0];
      powers[u] = *reinterpret_cast<const uint16_t*>(c.exponents + row + 2 * (at_lane & 15));
    }
  };
  float* const v_powers = reinterpret_cast<float*>(smem + kWaves * 2 * kTileBytes) + wave * 2 * kKeys;
  float* const v_scales = v_powers + kKeys;
  // Subtile u's powers of V (or 2^them) of the keys whose scores 4 j .. 4 j + 3 this lane holds.
  auto of_keys = [&](const float* from, int u, int j) {
    return *reinterpret_cast<const floatx4*>(from + 32 * u + 8 * j + 4 * (opaque(lane) >> 5));
  };
  auto weigh = [&](const floatx16& x, int u, V8 (&w)[2], float& l) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const floatx4 scale = of_keys(v_scales, u, 2 * h + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * h + 4 * j + i], a.scale_log2, -s.m));
          l += e;
          f[4 * j + i] = e * scale[i];
        }
      }
      w[h] = Num<T>::round8(f);
      if constexpr (D == 256) __builtin_amdgcn_sched_barrier(0);     // (eight at a time: registers)
    }
  };

  // (The two places as parameters that do not alias, as in narrow_piece.)
  auto tile = [&](int t, uint8_t* __restrict__ kt, uint8_t* __restrict__ vt) __attribute__((always_inline)) {
    uint32_t unmapped = 0;
#pragma unroll
    for (int h = 0; h < kGroups; ++h) unmapped |= page_of(t, h) < 0 ? 1u << h : 0u;
    const bool more = t + 1 < last;
    if (more && kGroups * (t + 1) - page_base >= 64) {
      page_base = kGroups * (t + 1);
      pages = load_group_pages(page_base);
    }
    // Loads end in order: V's kLoads came after K's (and the powers beside them, wherever
    // they stand among these), and below the next tile's K's after V's.
    wait_vmcnt<kLoads>();                   // K is there, V on its way
    asm volatile("" ::: "memory");
    const int here = opaque(lane);          // (places are found anew: registers)
    const int k_addr = (here & 31) * D + 16 * ((here >> 5) ^ k_code_swizzle<D>(here & 31));
    float k_scale[kSubs];
#pragma unroll
    for (int u = 0; u < kSubs; ++u) {
      k_scale[u] = scale_of(powers[u] & 0xFFu);
      if (here < 32) {
        constexpr ExponentRange kRange = exponent_range(std::is_same_v<T, __bf16> ? OSCAR_BF16 : OSCAR_FP16);
        constexpr uint32_t kLeast = 127 + kRange.low, kSpan = kRange.high - kRange.low;
        const uint32_t byte = powers[u] >> 8, v = byte - kLeast <= kSpan ? byte : kLeast;
        v_powers[32 * u + here] = (float)((int)v - 127);
        v_scales[32 * u + here] = scale_of(v);
      }
    }
    // (in this order at D = 256, kAhead reads ahead: left to it, the compiler asks for all
    // at once and spills registers)
    floatx16 x[kSubs];
    constexpr int kSteps = D / 32 * kSubs, kAhead = 2;
    auto k_codes = [&](int n) {
      return *reinterpret_cast<const u32x4*>(kt + n / (D / 32) * 32 * D + (opaque(k_addr) ^ (32 * (n % (D / 32)))));
    };
    u32x4 codes[kAhead];
    each<kAhead>([&](auto step) { codes[decltype(step)::value] = k_codes(decltype(step)::value); });
    if constexpr (D == 256) keep_order();
    each<kSteps>([&](auto step) {
      constexpr int n = decltype(step)::value, u = n / (D / 32), i = n % (D / 32);
      const V8 lower = operand_of<T>(u32x2{codes[n % kAhead][0], codes[n % kAhead][1]}, k_scale[u]);
      const V8 upper = operand_of<T>(u32x2{codes[n % kAhead][2], codes[n % kAhead][3]}, k_scale[u]);
      if constexpr (D == 256) keep_order();
      if constexpr (n + kAhead < kSteps) codes[n % kAhead] = k_codes(n + kAhead);
      x[u] = Num<T>::mfma(lower, s.q[2 * i], i == 0 ? floatx16{} : x[u]);
      x[u] = Num<T>::mfma(upper, s.q[2 * i + 1], x[u]);
      if constexpr (D == 256) keep_order();
    });
    asm volatile("" ::: "memory");
    if (more) {
      load_powers(t + 1);
      load_tile(t + 1, std::false_type{}, kt);
    }
    if constexpr (D == 256) keep_order();

    const int key0 = p.key0 + t * kKeys;
    const bool masked = !whole(key0) || unmapped != 0u;
    if (masked) {
#pragma unroll
      for (int u = 0; u < kSubs; ++u) mask_scores<16>(a, x[u], key0 + 32 * u, (unmapped >> (2 * u)) & 3u, here, s.pos);
    }
    if constexpr (D == 256) keep_order();
    V8 w[kSubs][2];
    float l = 0.f;
#pragma unroll
    for (int u = 0; u < kSubs; ++u) weigh(x[u], u, w[u], l);
    if constexpr (D == 256) keep_order();
    ushortx8 most = __builtin_bit_cast(ushortx8, w[0][0]);
    most = __builtin_elementwise_max(most, __builtin_bit_cast(ushortx8, w[0][1]));
#pragma unroll
    for (int u = 1; u < kSubs; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) most = __builtin_elementwise_max(most, __builtin_bit_cast(ushortx8, w[u][h]));
    uint16_t heaviest = 0;                  // (positive numbers compare as their bits do)
#pragma unroll
    for (int i = 0; i < 8; ++i) heaviest = max(heaviest, (uint16_t)most[i]);
    if (__ballot(heaviest > Num<T>::kMostBits)) {
      // A row is asked for its own heaviest weight: what becomes of it does not depend on
      // the other rows.
      float top = kNone;
#pragma unroll
      for (int u = 0; u < kSubs; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const floatx4 b = of_keys(v_powers, u, j);
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fmaf(x[u][4 * j + i], a.scale_log2, b[i]));
        }
      top = max_halves(top) - Num<T>::kLift;
      const bool over = max_halves(heaviest > Num<T>::kMostBits ? 1.f : 0.f) != 0.f && top > s.m;
      const float m = over ? top : s.m;
      const Lowered<true> f(s.m - m);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) s.acc[b] *= f.all;
      s.l = f.add(0.f, s.l);
      s.m = m;
      l = 0.f;
#pragma unroll
      for (int u = 0; u < kSubs; ++u) weigh(x[u], u, w[u], l);
    }
    s.l += l;

    if (more) wait_vmcnt<kLoads>();
    else wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    if (masked) special = take_out_nan<kTileBytes>(vt, here) || special;
    const int v_addr = v_code_read<D>(opaque(lane));
    keep_order();
    each<2 * kSubs * kBlocks>([&](auto step) {
      constexpr int h = decltype(step)::value / kBlocks, b = decltype(step)::value % kBlocks;
      s.acc[b] = Num<T>::mfma(operand_of<T>(v_codes_at(vt + h * 16 * D, opaque(v_addr) ^ (32 * b)), 1.f), w[h / 2][h % 2],
                              s.acc[b]);
      if constexpr (b % 4 == 3 || b == kBlocks - 1) keep_order();
    });
    asm volatile("" ::: "memory");
    if (more) load_tile(t + 1, std::true_type{}, vt);
  };
  uint8_t* const kt = smem + wave * 2 * kTileBytes;
  if (first < last) {
    load_powers(first);
    load_tile(first, std::false_type{}, kt);
    __builtin_amdgcn_sched_barrier(0);      // (the waits count K's loads before V's)
    load_tile(first, std::true_type{}, kt + kTileBytes);
  }
  for (int t = first; t < last; ++t) tile(t, kt, kt + kTileBytes);
  if (__builtin_expect(special, 0))
    for (int t = first; t < last; ++t) {
      const int key0 = p.key0 + t * kKeys;
      add_nan<T, D, kKeys>(a, c, p, key0, whole(key0), lane, s);
    }
  combine_waves<T, D, D == 256 ? 2 : 1, true>(a, p, s, smem, tid, lane, wave);
}

// ---------------------------------------------------------------- kernels
// (Codes past the caches, kOnce, where they are more than the last-level cache holds: 32
// users' token over 2K to 16K keys of 8 heads of 128, 578 MB, 123 us, through them 135; 32
// users' 4 of one head of 256, 146 MB, 39 us, through them 37; 48 rows over 32 MB 33, 31.
// At D = 64 neighbouring heads share lines, which L2 keeps for the second: 8 heads of 32
// users, 297 MB, 88 us, through them 82; of one head, 587 MB, 76 and 81.)
template <typename T, int D, int kPolicy>
__global__ __launch_bounds__(kThreads, kCodeWgs) void code_kernel(QuantChunkArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[code_lds(D)];
  code_piece<T, D, kPolicy>(a, a.wide.pieces[blockIdx.x], smem);
}
// A step with wide pieces, the narrow ones first where they are few, as mixed_kernel.
constexpr int kFewNarrow = kCus;
template <typename T, int D>
__global__ __launch_bounds__(kThreads, kWideWgs) void quant_kernel(QuantChunkArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[std::max(code_lds(D), wide_lds(D))];
  const int total = a.wide.narrow + a.wide.wide, lead = a.wide.narrow <= kFewNarrow ? 0 : a.wide.narrow;
  const int at = (int)blockIdx.x + lead, i = at < total ? at : at - total;
  if (i >= a.wide.narrow) wide_piece<T, D>(a.wide, a.wide.pieces[i], smem);
  else code_piece<T, D, kKept>(a, a.wide.pieces[i], smem);
}

// The sources' keys as 16-bit pages of 16 keys [K | V][key][head][D], a workgroup each,
// and the pages' block table.  A thread takes 8 codes at a time, four times at once.  Memory
// and a launch bound it: 24579 keys of a head of 256 7.8 us (38 MB, 4.8 TB/s), 12288 of 8
// heads of 128 15 (75 MB, 5.0 TB/s; the products over them then take 690).
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
// Rows of a request that are computed from codes, at most.  From codes / converted first,
// us: 8 users' 48 rows over 8000 keys, D = 256, 24 / 41; 4 users' 96 over 16000 30 / 45,
// 192 over 8000 32 / 39; 16 users' 64 over 4000, D = 128, 8 heads, 55 / 128; 8 users' 256
// over 2000, D = 64, 4 heads, 33 / 30, 192 of D = 128 72 / 87.
inline PlanRule quant_rule(int32_t head_size) {
  const int32_t rows = head_size == 64 ? 96 : 192;
  return PlanRule{head_size, rows, {kCus, 2 * kCus}, 1., 3 * kCus};
}

// The wide pieces' keys, table row by table row, and the pieces' table rows in the pages'.
void make_sources(Plan& plan, std::vector<Source>& sources, int64_t& pages) {
  struct Range {
    int32_t row, from, to;                  // groups of 16 keys
  };
  std::vector<Range> ranges;
  ranges.reserve(plan.wide.size());
  for (const Piece& p : plan.wide) {
    if (p.key0 < p.head_keys)
      ranges.push_back(Range{p.head_row, p.key0 / 16, (std::min(p.key1, p.head_keys) + 15) / 16});
    if (p.key1 > p.head_keys) ranges.push_back(Range{p.table_row, std::max(p.key0, p.head_keys) / 16, (p.key1 + 15) / 16});
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& x, const Range& y) { return x.row < y.row; });
  pages = 0;
  for (size_t i = 0; i < ranges.size();) {
    Range all = ranges[i];
    for (; i < ranges.size() && ranges[i].row == all.row; ++i) {
      all.from = std::min(all.from, ranges[i].from);
      all.to = std::max(all.to, ranges[i].to);
    }
    if (pages + all.to - all.from > INT32_MAX) throw 0;
    sources.push_back(Source{all.row, all.from, all.to - all.from, (int32_t)pages});
    pages += all.to - all.from;
  }
  auto base = [&](int32_t row) {            // of a row that none of the piece's keys are on: any
    const auto at = std::lower_bound(sources.begin(), sources.end(), row,
                                     [](const Source& x, int32_t y) { return x.table_row < y; });
    return at == sources.end() ? 0 : at->page0 - at->group0;
  };
  for (Piece& p : plan.wide) {
    p.table_row = base(p.table_row);
    p.head_row = p.head_keys > 0 ? base(p.head_row) : 0;
  }
}

// Narrow pieces that read the same lines (the row tiles of one request, and at D = 64, with
// two heads to a line, neighbouring heads) 8 workgroups apart, which is on one XCD, at one
// time: its L2 then gives both what was read for either.  (32 users' 4 tokens, 16 heads
// of 64 on 4, 2K to 16K keys: 60 us for 46.)
void order_pieces(std::vector<Piece>& pieces, int32_t head_size) {
  const int32_t heads = head_size == 64 ? 2 : 1;       // of a line
  if (heads == 1 && std::none_of(pieces.begin(), pieces.end(), [](const Piece& p) { return p.row0 > 0; })) return;
  // (a request's pieces stand together; of one they go by line and key, and then as before)
  std::vector<std::pair<uint64_t, uint32_t>> order(pieces.size());
  for (size_t i = 0; i < order.size(); ++i)
    order[i] = {(uint64_t)(uint32_t)(pieces[i].kv_head / heads) << 32 | (uint32_t)pieces[i].key0, (uint32_t)i};
  std::vector<uint32_t> groups{0};          // where they begin in the order
  for (size_t i = 0; i < order.size();) {
    size_t end = i + 1;
    auto of_one = [&](const Piece& p) { return p.table_row == pieces[i].table_row && p.token0 == pieces[i].token0; };
    while (end < order.size() && of_one(pieces[end])) ++end;
    std::sort(order.begin() + (std::ptrdiff_t)i, order.begin() + (std::ptrdiff_t)end);
    for (size_t k = i + 1; k <= end; ++k)
      if (k == end || order[k].first != order[k - 1].first) groups.push_back((uint32_t)k);
    i = end;
  }
  std::vector<Piece> to;
  to.reserve(pieces.size());
  for (size_t g = 0; g + 1 < groups.size(); g += 8) {
    const size_t end = std::min(g + 8, groups.size() - 1), before = to.size();
    const uint32_t all = groups[end] - groups[g];
    for (uint32_t m = 0; to.size() - before < all; ++m)
      for (size_t i = g; i < end; ++i)
        if (groups[i] + m < groups[i + 1]) to.push_back(pieces[order[groups[i] + m].second]);
  }
  pieces.swap(to);
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
  static_assert(kCodeWgs * code_lds(D) <= 160 * 1024 &&
                kWideWgs * std::max(code_lds(D), wide_lds(D)) <= 160 * 1024,
                "the workgroups of a CU must fit its 160 KiB of LDS");
  if (step.pages > 0) pages_kernel<T><<<step.pages, 256, 0, stream>>>(pages);
  const uint32_t pieces = (uint32_t)(step.chunk.narrow + step.chunk.wide);
  if (step.chunk.wide == 0 && step.once != 0) code_kernel<T, D, kOnce><<<pieces, kThreads, 0, stream>>>(a);
  else if (step.chunk.wide == 0) code_kernel<T, D, kKept><<<pieces, kThreads, 0, stream>>>(a);
  else quant_kernel<T, D><<<pieces, kThreads, 0, stream>>>(a);
  // (wide pieces' maxima are of scores alone: their joins are the plain cache's)
  return step.chunk.narrow > 0 ? launch_joins<T, D, true>(a.wide, step.chunk, stream)
                               : launch_joins<T, D, false>(a.wide, step.chunk, stream);
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
    order_pieces(plan.narrow, cache->head_size);
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
    int64_t codes = 0;                      // bytes that narrow pieces read
    for (const Piece& p : plan.narrow)
      if (p.row0 == 0) codes += 2ll * cache->head_size * (p.key1 - p.key0);
    const bool half_lines = cache->head_size == 64 && cache->num_kv_heads > 1 && cache->k_stride_head == 64;
    step->once = codes > kLastCache && !half_lines;
    step->reserved = 0;
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
  if (s.narrow < 0 || s.wide < 0 || s.few_joins < 0 || s.joins < s.few_joins || s.parts < 0 || s.join_rows < 0 ||
      s.join_rows > kTileRows || (s.joins > s.few_joins && s.join_rows == 0) || step->sources < 0 ||
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
