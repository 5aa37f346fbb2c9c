// The paged cache's address arithmetic (kv_view.h), on the host: every entry that is
// no page is told apart, every place lies inside its page and inside the cache,
// also where element offsets pass 32 bits.
#include <climits>
#include <cstdio>
#include <set>

#include "kv_view.h"

static int bad = 0;
#define CHECK(...) do { if (!(__VA_ARGS__)) { std::printf("line %d: %s\n", __LINE__, #__VA_ARGS__); ++bad; } } while (0)

int main() {
  using mit2hip::CacheView;
  const int32_t entries[] = {0, 3, 4, -1, INT_MAX, INT_MIN, 2, 5};
  for (int shift = 0; shift <= 10; ++shift) {
    const CacheView c = {nullptr, nullptr, entries, 4, shift, 3, 4};  // two sequences of four entries
    CHECK(c.capacity() == 4 << shift);
    for (int seq = 0; seq < 2; ++seq)
      for (int j = 0; j < c.capacity(); ++j) {
        const int e = entries[4 * seq + (j >> shift)];
        CHECK(c.page_of(seq, j) == (e >= 0 && e < 4 ? e : -1));
      }
    for (int D : {32, 96, 256}) {
      std::set<int64_t> at;
      for (int page = 0; page < 4; ++page)
        for (int h = 0; h < 3; ++h)
          for (int j = 5 << shift; j < 6 << shift; ++j) {
            const int64_t x = c.row_in(page, j, D) + h * c.head_stride(D);
            CHECK(x >= 0 && x + D <= (int64_t)4 * 3 * D << shift && x % D == 0 && at.insert(x).second);
          }
      CHECK(at.size() == (size_t)12 << shift);
    }
  }
  const CacheView big = {nullptr, nullptr, entries, INT_MAX, 10, 1024, 1 << 20};
  CHECK(big.page_of(0, 4 << 10) == -1);  // INT_MAX itself is past the last page
  CHECK(big.row_in(INT_MAX - 1, 1023, 256) == (((int64_t)(INT_MAX - 1) * 1024 << 10) + 1023) * 256);
  CHECK(big.capacity() == 1 << 30);
  std::printf("%d wrong\n", bad);
  return bad ? 1 : 0;
}
