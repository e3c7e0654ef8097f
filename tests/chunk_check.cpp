// Host check of csrc/kk_cache_index.h's cut of sequences into chunks: every
// step lies in one chunk, no sequence has more than its limit, and a batch
// never has more chunks than the grid that is launched for it.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "kk_cache_index.h"

using namespace kk;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: B %lld tokens %lld units %lld most %lld least %lld c %lld\n", __LINE__, \
    (long long)B, (long long)tokens, (long long)units, (long long)most, (long long)least, (long long)c); return 1; } } while (0)

int main() {
  for (int round = 0; round < 20000; ++round) {
    const int64_t B = 1 + rand() % 200, tokens = rand() % 3 ? rand() % 5000 : rand() % 4000000;
    const int64_t units = 1 + rand() % 1000, most = units + rand() % 3 * (rand() % 4000), least = 1 + rand() % 16;
    std::vector<int64_t> steps(B);
    int64_t total = 0, c = 0;
    for (auto& n : steps) {  // (a window's first step may start up to a step before its first token)
      const int64_t seen = rand() % 4 ? rand() % (tokens + 1) : tokens, lead = rand() % kStep;
      n = seen ? (seen + lead + kStep - 1) / kStep : 0;
      total += n;
    }
    c = chunk_size(total, units, most, least);
    int64_t chunks = 0;
    for (int64_t n : steps) {
      const int64_t count = chunk_count(n, c), each = chunk_steps(n, c);
      CHECK(count >= 1 && count <= kMaxChunks);
      CHECK(count * each >= n && (count == 1 || (count - 1) * each < n));
      chunks += count;
    }
    CHECK(c >= least && chunks <= grid_chunks(B, tokens, most, least));
  }
  std::puts("ok");
}
