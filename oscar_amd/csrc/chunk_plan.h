// How a step of the chunk attention is cut into pieces, on the host.
#pragma once

#include "chunk_pieces.h"
#include "row_span.h"

#include <algorithm>
#include <cstddef>
#include <cstring>
#include <vector>

namespace oscar {
namespace {

struct Plan {
  std::vector<Piece> narrow, wide;
  std::vector<Join> joins;
  std::vector<SharedPart> parts;
  int32_t slots = 0;
};

// Keys [0, keys) that requests first .. first + count - 1 begin with, computed for all
// their rows as if they were one request's.
struct Prefix {
  int32_t first, count, keys;
};
// The rows of a prefix and kv head, 32 to a slot, in pieces that all have the same keys.
struct PrefixRows {
  int32_t slot0 = -1, groups = 0, pieces = 0;
};

// What a cache asks of the plan.
struct PlanRule {
  int32_t head_size;
  int32_t narrow_rows;     // of a request and kv head, at most
  int32_t resident[2];     // narrow pieces that read at full rate, and that fit the GPU at once
  double key_bytes;        // of a key's features, read
  int32_t uneven;          // narrow pieces to cut very uneven row tiles to, where they fill the GPU; 0: never
};
inline PlanRule plain_rule(int32_t head_size) {
  // Up to 32 rows a request is narrow (28 rows of 16 users over 1000 keys, D = 128: 20.4
  // us, as wide tiles 24.2; 30 of 8 users over 16000, D = 256, 31.1, 30.1), from 33 on
  // wide, where narrow tiles would read its keys twice (48 rows, the same: 24.7 us, as
  // narrow 23.2; 32.2, 36.1; 32 users over 4000 32.5, 49.6).
  return PlanRule{head_size, kTileRows, {kCus, kCus * narrow_wgs(head_size)}, 2., 0};
}

struct RowTile {
  Piece piece;
  int32_t tiles;           // of 32 keys
  int32_t of_prefix = -1;  // PrefixRows that it is some of
  int32_t with_prefix = -1, prefix_row = 0;      // PrefixRows that its rows go on from, and where they begin there
};

// What a request has of a prefix: its rows go on from row `row` of PrefixRows `with` (of its
// first kv head), or, without (-1), it computes the keys itself, on table row `head`.
struct OfPrefix {
  int32_t keys = 0, with = -1, row = 0, head = 0;
};

// The row tiles of a request, `rows` rows each, with the keys that they see, but for those of a
// prefix that it goes on from.
void row_tiles(int32_t token0, int32_t n, int32_t seq, int32_t table_row, int32_t group, int32_t kv_heads,
               int32_t window, int32_t rows, const OfPrefix& prefix, std::vector<RowTile>& out) {
  const int32_t all = n * group;
  for (int32_t r = 0; r < all; r += rows) {
    Piece p{};
    p.token0 = token0;
    p.pos0 = seq - n;
    p.table_row = table_row;
    p.row0 = r;
    p.rows = std::min(rows, all - r);
    p.slot = -1;
    if (prefix.with < 0 && prefix.head != table_row) {
      p.head_keys = prefix.keys;
      p.head_row = prefix.head;
    }
    const int32_t lo = window > 0 ? std::max(0, p.pos0 + r / group - window + 1) : prefix.with >= 0 ? prefix.keys : 0;
    p.key0 = lo / kTileKeys * kTileKeys;
    p.key1 = p.pos0 + (r + p.rows - 1) / group + 1;
    for (int32_t h = 0; h < kv_heads; ++h) {
      p.kv_head = h;
      RowTile x{p, (p.key1 - p.key0 + kTileKeys - 1) / kTileKeys};
      if (prefix.with >= 0) {
        x.with_prefix = prefix.with + h;
        x.prefix_row = prefix.row + r;
      }
      out.push_back(x);
    }
  }
}

// The row tiles of a prefix: all rows of `tokens` tokens from token0 on, which see all
// of its keys.
void prefix_tiles(int32_t token0, int32_t tokens, int32_t keys, int32_t table_row, int32_t group, int32_t kv_heads,
                  int32_t rows, int32_t of_prefix, std::vector<RowTile>& out) {
  const int32_t all = tokens * group;
  for (int32_t r = 0; r < all; r += rows)
    for (int32_t h = 0; h < kv_heads; ++h) {
      RowTile x{Piece{token0, keys, table_row, h, r, std::min(rows, all - r), 0, keys, -1, 0, 0, 0}, keys / kTileKeys};
      x.of_prefix = of_prefix + h;
      out.push_back(x);
    }
}

// Whether a row tile in n pieces leaves partials.
bool leaves_partials(const RowTile& x, int32_t n) { return n > 1 || x.of_prefix >= 0 || x.with_prefix >= 0; }

// A row tile in n pieces of equal length, but for a key tile.
void cut(const RowTile& x, int32_t n, Plan& plan, std::vector<PrefixRows>& prefixes, std::vector<Piece>& out) {
  if (!leaves_partials(x, n)) {
    out.push_back(x.piece);
    return;
  }
  const int32_t groups = (x.piece.rows + kTileRows - 1) / kTileRows;
  int32_t slot = plan.slots, step = groups;
  if (x.of_prefix >= 0) {                   // (the join's rows are the requests')
    PrefixRows& rows = prefixes[x.of_prefix];
    if (rows.slot0 < 0) {
      rows.slot0 = plan.slots;
      rows.pieces = n;
      plan.slots += n * rows.groups;
    }
    slot = rows.slot0 + x.piece.row0 / kTileRows;
    step = rows.groups;
  } else {
    plan.slots += n * groups;
    for (int32_t g = 0; g < groups; ++g) {
      if (x.with_prefix >= 0) plan.parts.push_back(SharedPart{x.with_prefix, 0, 0, x.prefix_row + g * kTileRows});
      plan.joins.push_back(Join{x.piece.token0, x.piece.kv_head, x.piece.row0 + g * kTileRows,
                                std::min(kTileRows, x.piece.rows - g * kTileRows), slot + g, step, n,
                                x.with_prefix >= 0 ? (int32_t)plan.parts.size() : 0});
    }
  }
  for (int32_t s = 0; s < n; ++s) {
    Piece p = x.piece;
    p.key0 = x.piece.key0 + kTileKeys * (int32_t)((int64_t)x.tiles * s / n);
    p.key1 = std::min<int32_t>(x.piece.key1, x.piece.key0 + kTileKeys * (int32_t)((int64_t)x.tiles * (s + 1) / n));
    p.slot = slot + s * step;
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
// `uneven`: where the longest piece is still more than twice a resident piece's mean length
// and 32 key tiles above it, as with as many row tiles or nearly as many, all are cut to so
// many mean lengths.
// 8-bit caches, whole / cut to three a CU, us: 64 users over 100 to 16000 keys, D = 128,
// 8 kv heads, 195 / 107, 128 users 291 / 203, 4 tokens of 128 users, D = 64, 4 heads,
// 155 / 84; 256 over 100 to 8000, D = 256, 175 / 103; 300 over 1000 and one over 60000
// 954 / 90, 508 over 1000 and one 257 / 76, 490 77 / 75; 62 and one of 8 heads, D = 128, 328 /
// 57; 168 and one beside a prompt of 1200 482 / 56; without the second condition 256 over 100
// to 800 27 / 32.
constexpr int32_t kMuchLonger = 32;
void plan_narrow(const std::vector<RowTile>& rows, const PlanRule& rule, double beside, Plan& plan,
                 std::vector<PrefixRows>& prefixes) {
  int64_t total = 0;
  int32_t most = 0;
  for (const RowTile& x : rows) {
    total += x.tiles;
    most = std::max(most, x.tiles);
  }
  const int32_t uncut = rule.head_size == 256 ? 8 : 16;
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
  const bool reading = total * rule.key_bytes > 2 * 240 * beside;
  int64_t resident = beside == 0. ? rule.resident[0] : reading ? 2 * kCus : 2 * kCus / 3;
  int64_t per = fit(resident);
  if (beside == 0. && ((int64_t)rows.size() >= rule.resident[0] || 100 * per * rule.resident[0] > 115 * total)) {
    resident = rule.resident[1];
    per = fit(resident);
  }
  const int64_t mean = std::max<int64_t>(kWaves, (total + resident - 1) / resident);
  const int64_t longest = std::min<int64_t>(per, most);
  if (rule.uneven > 0 && longest > 2 * mean && longest > mean + kMuchLonger)
    per = std::max<int64_t>(kWaves, (total + rule.uneven - 1) / rule.uneven);
  for (const RowTile& x : rows) cut(x, pieces_of(x, per), plan, prefixes, plan.narrow);
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
double plan_wide(const std::vector<RowTile>& rows, int32_t head_size, Plan& plan, std::vector<PrefixRows>& prefixes) {
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
      cuts = cuts || leaves_partials(x, n);
      count[(x.tiles + n - 1) / n + (leaves_partials(x, n) ? kCutCost : kPieceCost)] += n;
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
  for (const RowTile& x : rows) cut(x, pieces_of(x, per), plan, prefixes, plan.wide);
  std::stable_sort(plan.wide.begin(), plan.wide.end(),
                   [](const Piece& x, const Piece& y) { return x.key1 - x.key0 > y.key1 - y.key0; });
  // The first two rounds of workgroups share CUs in order: the longest pieces,
  // shortest first, meet the next ones, longest first.
  std::reverse(plan.wide.begin(), plan.wide.begin() + (std::ptrdiff_t)std::min<size_t>(kCus, plan.wide.size()));
  return best;
}

// Where a step has rows for a wide piece a CU, its row tiles are not cut and the matrix unit
// bounds them.  Of a prefix it then has the same products to do either way, but for the rows
// that a request's last tile lacks, which the prefix' tiles have; sharing costs partials, of
// the prefix and of the request's own keys: 16 (D + 2) bytes a row, written and read, take as
// long at 5 TB/s as 4 D flops a key of 800 keys at 1 PFLOP/s.  So a request whose idle rows
// times the prefix' keys are less than 800 times its rows computes them itself, from the first
// one's table row.  Shared / each for itself, us: 8 prompts of 4096 tokens over 1024 keys, 32
// heads of 128 on 8, 1933 and 1.09 GB of partials / 1571 and none; 16 of 2048 over 64 1032 /
// 660; 8 of 300 over 960 79 / 65; 32 of 32 over 64 24 / 10.5, over 1024 41 / 29; 128 of 16
// over 64 44 / 21, but over 1024 72 / 81; 128 of 10 over 1024 55 / 79; 8 of 1200 over 4096, 6
// heads of 256 on one, 273 / 254; of the 8-bit cache (the keys converted once for all) 32 of 64
// over 4096 167 / 146.  With fewer rows tiles are cut in any case: 4 of 512 over 24576, D =
// 256, 292 / 305, 8 of 300 over 1024 52 / 45, 16 of 16 over 8192, D = 128, 52 / 73.
// The requests between such are computed together, as far as they follow each other.
constexpr int64_t kKeysOfPartial = 800;
void make_plan(const int32_t* qsl, const int32_t* seqs, int32_t num_requests, int32_t group, int32_t kv_heads,
               const PlanRule& rule, int32_t window, const std::vector<Prefix>& shared, Plan& plan) {
  std::vector<RowTile> narrow, wide;
  std::vector<PrefixRows> prefixes;
  auto rows_of = [&](int32_t i) { return (int64_t)(qsl[i + 1] - qsl[i]) * group; };
  int64_t wide_rows = 0;
  if (!shared.empty())
    for (int32_t i = 0; i < num_requests; ++i)
      if (rows_of(i) > rule.narrow_rows) wide_rows += rows_of(i) * kv_heads;
  auto prefix = shared.begin();
  OfPrefix of;                              // the prefix that request i begins with,
  int32_t until = 0, together = 0, first_token = 0;    // and its requests up to `together` that share it
  auto alone = [&](int32_t i) {
    const int64_t rows = rows_of(i), idle = (kWideRows - rows % kWideRows) % kWideRows;
    return wide_rows >= (int64_t)kCus * kWideRows && rows > rule.narrow_rows && of.keys * idle < kKeysOfPartial * rows;
  };
  for (int32_t i = 0; i < num_requests; ++i) {
    const int32_t n = qsl[i + 1] - qsl[i];
    if (i >= until) of = OfPrefix{};
    if (prefix != shared.end() && i == prefix->first) {
      of.keys = prefix->keys;
      until = i + prefix->count;
      together = i;
      of.head = i;                          // a request's that has tokens
      while (qsl[of.head + 1] == qsl[of.head]) ++of.head;
      ++prefix;
    }
    if (of.keys > 0 && i >= together) {
      int32_t members = 0;
      for (; together < until && !alone(together); ++together) members += qsl[together + 1] > qsl[together];
      of.with = -1;
      if (members > 1) {
        of.with = (int32_t)prefixes.size();
        first_token = qsl[i];
        const int32_t tokens = qsl[together] - qsl[i];
        PrefixRows rows;
        rows.groups = (tokens * group + kTileRows - 1) / kTileRows;
        prefixes.insert(prefixes.end(), kv_heads, rows);
        if (tokens * (int64_t)group <= rule.narrow_rows)
          prefix_tiles(qsl[i], tokens, of.keys, of.head, group, kv_heads, kTileRows, of.with, narrow);
        else
          prefix_tiles(qsl[i], tokens, of.keys, of.head, group, kv_heads, kWideRows, of.with, wide);
      }
      together = std::max(together, i + 1);
    }
    of.row = of.with >= 0 ? (qsl[i] - first_token) * group : 0;
    if (rows_of(i) <= rule.narrow_rows)
      row_tiles(qsl[i], n, seqs[i], i, group, kv_heads, window, kTileRows, of, narrow);
    else
      row_tiles(qsl[i], n, seqs[i], i, group, kv_heads, window, kWideRows, of, wide);
  }
  const double beside = wide.empty() ? 0. : plan_wide(wide, rule.head_size, plan, prefixes);
  if (!narrow.empty()) plan_narrow(narrow, rule, beside, plan, prefixes);
  for (SharedPart& p : plan.parts) {
    const PrefixRows& rows = prefixes[p.slot0];
    p = SharedPart{rows.slot0, rows.groups, rows.pieces, p.row};
  }
  std::stable_partition(plan.joins.begin(), plan.joins.end(), [&](const Join& j) {
    return j.count + (j.shared > 0 ? plan.parts[j.shared - 1].count : 0) <= kFewParts;
  });
}

// ---------------------------------------------------------------- the step
// A step's arguments.  *pages: of the block table, in pages of block_size.
int check_step(const int32_t* qsl, const int32_t* seqs, int32_t num_requests, int32_t num_heads, int32_t num_kv_heads,
               int32_t window, int32_t block_size, int32_t* pages) {
  if (num_requests < 0 || (num_requests > 0 && (qsl == nullptr || seqs == nullptr)) || num_heads < 1 ||
      num_heads % num_kv_heads || num_heads > (1 << 16) || window < 0)
    return kErrInvalidArgument;
  const int32_t group = num_heads / num_kv_heads;
  *pages = 0;
  for (int32_t i = 0; i < num_requests; ++i) {
    const int64_t n = (int64_t)qsl[i + 1] - qsl[i];
    if (qsl[i] < 0 || n < 0 || seqs[i] < n || n * group > kMostKeys || seqs[i] > kMostKeys) return kErrInvalidArgument;
    if (n > 0) *pages = std::max(*pages, (seqs[i] - 1) / block_size + 1);
  }
  return kOk;
}

// Prefixes in the order of their requests, whole key tiles of them (what is left a request
// reads with its own keys), without those of less than two requests with tokens.
int check_prefixes(const oscar_prefix* prefixes, int32_t count, const int32_t* qsl, const int32_t* seqs,
                   int32_t num_requests, int32_t group, int32_t window, std::vector<Prefix>& out) {
  if (count < 0 || (count > 0 && (prefixes == nullptr || window > 0))) return kErrInvalidArgument;
  int32_t until = 0;
  for (int32_t i = 0; i < count; ++i) {
    const oscar_prefix& p = prefixes[i];
    if (p.first < until || p.requests < 0 || p.keys < 0 || p.requests > num_requests - p.first) return kErrInvalidArgument;
    until = p.first + p.requests;
    int32_t with_tokens = 0;
    for (int32_t r = p.first; r < until; ++r) {
      const int32_t n = qsl[r + 1] - qsl[r];
      if (n == 0) continue;
      ++with_tokens;
      if (p.keys > seqs[r] - n) return kErrInvalidArgument;
    }
    const int64_t rows = ((int64_t)qsl[until] - qsl[p.first]) * group;
    if (rows > kMostKeys) return kErrInvalidArgument;
    if (with_tokens > 1 && p.keys >= kTileKeys) out.push_back(Prefix{p.first, p.requests, p.keys / kTileKeys * kTileKeys});
  }
  return kOk;
}

// Sizes of a plan, and its items: pieces, joins, prefix parts.
int pack_plan(const Plan& plan, int32_t head_size, void* items, size_t items_size, oscar_chunk_step* step) {
  if (plan.narrow.size() + plan.wide.size() > INT32_MAX || plan.joins.size() > INT32_MAX) return kErrInvalidArgument;
  step->narrow = (int32_t)plan.narrow.size();
  step->wide = (int32_t)plan.wide.size();
  step->joins = (int32_t)plan.joins.size();
  step->parts = (int32_t)plan.parts.size();
  auto few = [&](const Join& j) { return j.count + (j.shared > 0 ? plan.parts[j.shared - 1].count : 0) <= kFewParts; };
  step->few_joins = (int32_t)std::count_if(plan.joins.begin(), plan.joins.end(), few);
  step->join_rows = 0;
  for (const Join& j : plan.joins)
    if (!few(j)) step->join_rows = std::max(step->join_rows, j.rows);
  const void* const from[4] = {plan.narrow.data(), plan.wide.data(), plan.joins.data(), plan.parts.data()};
  const size_t size[4] = {plan.narrow.size() * sizeof(Piece), plan.wide.size() * sizeof(Piece),
                          plan.joins.size() * sizeof(Join), plan.parts.size() * sizeof(SharedPart)};
  step->items_size = (int64_t)(size[0] + size[1] + size[2] + size[3]);
  step->workspace_size = (int64_t)plan.slots * kTileRows * (head_size + 2) * 4;
  if (items == nullptr) return kOk;
  if ((int64_t)items_size < step->items_size) return kErrWorkspaceTooSmall;
  uint8_t* to = static_cast<uint8_t*>(items);
  for (int i = 0; i < 4; ++i) {
    if (size[i] > 0) std::memcpy(to, from[i], size[i]);
    to += size[i];
  }
  return kOk;
}

// A plan's arguments that go by the step, the rows and the items; what a cache adds is
// left to the caller.
int step_args(const oscar_chunk_step* step, const void* items, const int32_t* block_table, int64_t block_table_stride,
              const oscar_heads* query, const oscar_heads* out, float scale, void* workspace, size_t workspace_size,
              int64_t need, ChunkArgs& a) {
  if (items == nullptr || block_table == nullptr || query->data == nullptr || out->data == nullptr ||
      block_table_stride < step->table_cols)
    return kErrInvalidArgument;
  if ((int64_t)workspace_size < need || (need > 0 && workspace == nullptr)) return kErrWorkspaceTooSmall;
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
                     2 * step->head_size};
  const RowSpan to{(uint64_t)(uintptr_t)a.out, a.out_token, a.out_head, step->num_tokens, step->num_heads,
                   2 * step->head_size};
  if (!same_rows(from, to) && !rows_apart(from, to)) return kErrOverlap;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.pieces = static_cast<const Piece*>(items);
  a.narrow = step->narrow;
  a.wide = step->wide;
  a.few_joins = step->few_joins;
  a.join_rows = step->join_rows;
  a.joins = reinterpret_cast<const Join*>(a.pieces + step->narrow + step->wide);
  a.parts = reinterpret_cast<const SharedPart*>(a.joins + step->joins);
  a.partials = static_cast<float*>(workspace);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.group = step->num_heads / step->num_kv_heads;
  a.block_size = step->block_size;
  a.window = step->window;
  a.group_div = make_fast_div((uint32_t)a.group);
  a.block_div = make_fast_div((uint32_t)a.block_size);
  return kOk;
}

template <typename T, int D, bool kPowers>
int launch_joins(const ChunkArgs& a, const oscar_chunk_step& step, hipStream_t stream) {
  const int64_t blocks = (int64_t)step.few_joins * (D / 32) + (int64_t)(step.joins - step.few_joins) * (step.join_rows * (D / 64));
  if (blocks > INT32_MAX) return kErrInvalidArgument;
  if (blocks > 0 && step.parts == 0) join_kernel<T, D, false, kPowers><<<(uint32_t)blocks, 256, 0, stream>>>(a);
  else if (blocks > 0) join_kernel<T, D, true, kPowers><<<(uint32_t)blocks, 256, 0, stream>>>(a);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace
}  // namespace oscar
