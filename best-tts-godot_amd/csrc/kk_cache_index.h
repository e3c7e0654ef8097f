// Which rows of which page a call to a paged cache touches: whole-number
// rules shared by the kernels and the host, safe for any values a caller's
// device memory may hold (negative or huge starts, counts and lengths).
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define KK_HD __attribute__((host, device)) inline __attribute__((always_inline))
#else
#define KK_HD inline
#endif

namespace kk {

// Rows of one page: `rows` new tokens (0: none) from `token` on, behind
// `held` rows that the page holds already; the page is the table's `column`.
struct PageRows {
  int rows, held, token;
  int64_t column;
};

// The j-th page that `count` (of at most T) tokens after `start` reach, in a
// sequence of `columns` pages of `block` rows.  Tokens past the last column
// are dropped.  0 <= held, held + rows <= block, 0 <= token and token + rows
// <= T, 0 <= column < columns whenever rows > 0.
KK_HD PageRows page_rows(int64_t start, int64_t count, int64_t T, int64_t block, int64_t columns, int64_t j) {
  PageRows r = {0, 0, 0, 0};
  if (start < 0 || start >= columns * block) return r;
  if (count > T) count = T;
  if (count > columns * block - start) count = columns * block - start;
  const int64_t column = start / block + j;
  const int64_t lo = j == 0 ? start : column * block;
  int64_t hi = (column + 1) * block;
  if (hi > start + count) hi = start + count;
  if (hi <= lo) return r;
  r.rows = static_cast<int>(hi - lo);
  r.held = static_cast<int>(lo - column * block);
  r.token = static_cast<int>(lo - start);
  r.column = column;
  return r;
}

// Tokens [lo, hi) of a cache that the query at `place` of its sequence sees:
// those up to itself, of a window of the last `window` (0: all), within what
// the table can hold.  Empty where place < 0.
struct Seen {
  int64_t lo, hi;
};
KK_HD Seen seen_tokens(int64_t place, int64_t window, int64_t capacity) {
  Seen s;
  s.hi = place < capacity ? place + 1 : capacity;
  s.lo = window > 0 && place >= window ? place - window + 1 : 0;
  if (s.hi < 0) s.hi = 0;
  if (s.lo > s.hi) s.lo = s.hi;
  return s;
}

// Long sequences cut into chunks over blocks (kk_attention.h).  A sequence of
// `steps` steps has chunk_count chunks of chunk_steps each; chunk_size is the
// size for a batch of `total` steps: `units` chunks of it, or, once those pass
// kLongChunk steps, `most`; `least` steps at least.  At most kMaxChunks a sequence.
constexpr int kStep = 64;        // tokens
constexpr int kLongChunk = 64;   // steps
constexpr int kMaxChunks = 64;   // a wave of the block that joins them has a lane for each
KK_HD int64_t chunk_size(int64_t total, int64_t units, int64_t most, int64_t least) {
  int64_t c = (total + units - 1) / units;
  if (c > kLongChunk && most > units) {
    c = (total + most - 1) / most;
    c = c < kLongChunk ? kLongChunk : c;
  }
  return c < least ? least : c;
}
KK_HD int64_t chunk_steps(int64_t steps, int64_t c) {
  const int64_t fewest = (steps + kMaxChunks - 1) / kMaxChunks;
  return c < fewest ? fewest : c;
}
KK_HD int64_t chunk_count(int64_t steps, int64_t c) {
  const int64_t each = chunk_steps(steps, c);
  return steps <= each ? 1 : (steps + each - 1) / each;
}
// What B sequences of at most `tokens` seen tokens each come to at the most
// (their first step may hold tokens that a window has left behind).
KK_HD int64_t grid_chunks(int64_t B, int64_t tokens, int64_t most, int64_t least) {
  const int64_t by_length = B * (tokens / kStep / least + 2);
  return by_length < B + most ? by_length : B + most;
}

}  // namespace kk
