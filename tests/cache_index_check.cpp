// Host check of csrc/kk_cache_index.h: random and extreme starts, counts,
// lengths and windows never name a row, token or column out of range, and
// together they name each wanted token once.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "kk_cache_index.h"

static int64_t pick() {
  static const int64_t odd[] = {0, 1, -1, 15, 16, 17, INT64_MAX, INT64_MIN, INT64_MAX - 1, 1LL << 40, -(1LL << 40)};
  const int r = rand();
  return r % 5 == 0 ? odd[rand() % 11] : rand() % 200;
}

#define CHECK(c) do { if (!(c)) { std::printf("line %d: start %lld count %lld T %lld block %lld columns %lld\n", \
    __LINE__, (long long)start, (long long)count, (long long)T, (long long)block, (long long)columns); return 1; } } while (0)

int main() {
  const int64_t blocks[] = {16, 32, 64, 128, 256};
  for (int i = 0; i < 2000000; ++i) {
    const int64_t start = pick(), count = pick(), T = 1 + rand() % 180, block = blocks[rand() % 5], columns = rand() % 12;
    const int64_t reach = (T + block - 2) / block + 1;
    int64_t next = 0;
    for (int64_t j = 0; j < reach; ++j) {
      const kk::PageRows r = kk::page_rows(start, count, T, block, columns, j);
      if (r.rows <= 0) continue;
      CHECK(r.held >= 0 && r.held + r.rows <= block && r.token == next && r.token + r.rows <= T);
      CHECK(r.column >= 0 && r.column < columns && r.column * block + r.held == start + r.token);
      next = r.token + r.rows;
    }
    int64_t want = count < T ? count : T;
    if (want < 0 || start < 0 || start >= columns * block) want = 0;
    if (want > 0 && want > columns * block - start) want = columns * block - start;
    CHECK(next == want);
    const int64_t window = llabs(count) == INT64_MIN ? 0 : (count < 0 ? 0 : count);
    const kk::Seen s = kk::seen_tokens(start, window, columns * block);
    CHECK(s.lo >= 0 && s.lo <= s.hi && s.hi <= columns * block);
    for (int64_t p = 0; p < columns * block; ++p) {
      const bool in = p <= start && (window == 0 || p > start - window);
      CHECK(in == (p >= s.lo && p < s.hi));
    }
  }
  std::printf("ok\n");
  return 0;
}
