// How a step of the chunk attention is cut into pieces, on the host.
#pragma once

#include "chunk_pieces.h"

#include <algorithm>
#include <cstddef>
#include <vector>

namespace oscar {
namespace {

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

}  // namespace
}  // namespace oscar
