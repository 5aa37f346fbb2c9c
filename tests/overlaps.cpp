// overlap.h against every pair of pieces, over small sets of all kinds: apart,
// slices of one buffer, interleaved, nested either way, broadcast, shifted by a
// part of a piece; and at strides where 64-bit byte offsets would wrap.
#include <cstdio>
#include <random>

#include "overlap.h"

using mit2hip::Pieces;

static bool hit(const Pieces& a, uint64_t ra, uint64_t ha, const Pieces& b, uint64_t rb, uint64_t hb) {
  const __int128 x = (__int128) reinterpret_cast<uintptr_t>(a.at) + (__int128)(ra * a.row + ha * a.head),
                 y = (__int128) reinterpret_cast<uintptr_t>(b.at) + (__int128)(rb * b.row + hb * b.head);
  return x < y + b.bytes && y < x + a.bytes;
}
static bool any(const Pieces& a, const Pieces& b, bool own) {
  for (uint32_t ra = 0; ra < a.rows; ++ra)
    for (uint32_t ha = 0; ha < a.heads; ++ha)
      for (uint32_t rb = 0; rb < b.rows; ++rb)
        for (uint32_t hb = 0; hb < b.heads; ++hb)
          if (!(own && ra == rb && ha == hb) && hit(a, ra, ha, b, rb, hb)) return true;
  return false;
}

int main() {
  std::mt19937 rng(1);
  auto pick = [&](uint32_t lo, uint32_t hi) { return lo + rng() % (hi - lo + 1); };
  int wrong = 0, yes = 0, no = 0;
  for (int t = 0; t < 200000; ++t) {
    const uint32_t D = pick(1, 4), size = pick(0, 1) ? 2 : 4;
    auto set = [&](uintptr_t base) {
      const uint32_t rows = pick(0, 5), heads = pick(1, 5);
      uint64_t head = D * pick(0, 4) + pick(0, 1), row = pick(0, 2) ? heads * D * pick(1, 4) : D * pick(0, 12) + pick(0, 1);
      if (pick(0, 3) == 0) std::swap(row, head);
      return mit2hip::pieces(reinterpret_cast<void*>(base), row, head, rows, heads, D, size);
    };
    Pieces a = set(4096), b = set(4096 + size * pick(0, 40) - (pick(0, 3) ? 0 : size * pick(0, 60)));
    if (pick(0, 1)) { b.row = a.row; if (pick(0, 1)) b.head = a.head; }
    const bool self = any(a, a, true), both = any(a, b, false);
    (both ? yes : no) += 1;
    if (mit2hip::meet_themselves(a) != self) ++wrong;
    if (mit2hip::meet(a, b) != both || mit2hip::meet(b, a) != both) ++wrong;
    const uint64_t n = a.rows * a.bytes, m = b.heads * b.bytes;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    if (mit2hip::meet(a.at, n, b.at, m) != (n && m && x < y + m && y < x + n)) ++wrong;
  }
  // a row stride whose second row's byte offset is 2^64 + 64: far away, not on the first
  const Pieces far = mit2hip::pieces(reinterpret_cast<void*>(4096), (1ull << 62) + 16, 64, 2, 2, 64, 4);
  if (mit2hip::meet_themselves(far)) ++wrong;
  // a projection's rows: queries turned in place beside their keys, 16,777,215 rows of 64 heads
  const uint64_t width = (64 + 2 * 8) * 128;
  char* const base = reinterpret_cast<char*>(1 << 20);
  const Pieces q = mit2hip::pieces(base, width, 128, (1u << 24) - 1, 64, 128, 2), k = mit2hip::pieces(base + 64 * 128 * 2, width, 128, (1u << 24) - 1, 8, 128, 2);
  if (mit2hip::meet(q, k) || mit2hip::meet_themselves(q) || !mit2hip::meet(q, q)) ++wrong;
  std::printf("%d wrong of %d that meet, %d that do not\n", wrong, yes, no);
  return wrong ? 1 : 0;
}
