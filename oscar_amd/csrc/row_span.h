// Where a call's rows lie, and whether two kinds of them share memory.
#pragma once

#include <stdint.h>

#include <numeric>

namespace oscar {

// tokens x heads rows of `row` bytes; strides in bytes, not negative (of axes of one
// entry: 0).
struct RowSpan {
  uint64_t at;
  int64_t token, head, tokens;
  int32_t heads;
  int64_t row;
};

inline bool same_rows(const RowSpan& x, const RowSpan& y) {
  return x.at == y.at && x.token == y.token && x.head == y.head && x.heads == y.heads;
}

// Patterns x_width and y_width wide, `delta` apart, that repeat with `period`: side by side?
inline bool beside(__int128 delta, int64_t period, __int128 x_width, __int128 y_width) {
  if (period == 0) return false;
  const __int128 rest = delta % period, at = rest < 0 ? rest + period : rest;
  return at >= x_width && at + y_width <= period;
}

// Whether the rows share no memory: told from their ranges, or, for slices of one
// projection, from where they lie in its tokens, heads or rows.  Layouts more tangled
// than that count as sharing.
inline bool rows_apart(const RowSpan& x, const RowSpan& y) {
  if (x.tokens < 1 || x.heads < 1 || y.tokens < 1 || y.heads < 1) return true;
  const __int128 delta = (__int128)y.at - (__int128)x.at;
  const __int128 x_token = (__int128)(x.tokens - 1) * x.token, x_head = (__int128)(x.heads - 1) * x.head;
  const __int128 y_token = (__int128)(y.tokens - 1) * y.token, y_head = (__int128)(y.heads - 1) * y.head;
  if (delta >= x_token + x_head + x.row || -delta >= y_token + y_head + y.row) return true;
  if (x.token == y.token && beside(delta, x.token, x_head + x.row, y_head + y.row)) return true;
  if (x.head == y.head && beside(delta, x.head, x_token + x.row, y_token + y.row)) return true;
  return beside(delta, std::gcd(std::gcd(x.token, x.head), std::gcd(y.token, y.head)), x.row, y.row);
}

}  // namespace oscar
