// overlap.h -- whether an operator's buffers lie on one another, from their
// addresses, strides and counts alone (host; no HIP).
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace mit2hip {

// rows x heads pieces of `bytes` each; strides in bytes.
struct Pieces {
  const void* at;
  unsigned __int128 row, head;
  uint32_t rows, heads;
  uint64_t bytes;
};
inline Pieces pieces(const void* at, uint64_t row, uint64_t head, uint32_t rows, uint32_t heads, uint32_t dim, size_t elem) {
  return {at, (unsigned __int128)row * elem, (unsigned __int128)head * elem, rows, heads, (uint64_t)dim * elem};
}

namespace overlap {
typedef __int128 i128;
inline i128 address(const void* p) { return (i128) reinterpret_cast<uintptr_t>(p); }

// A set as an outer and an inner stride (the larger outside), without those of a single piece.
struct Nest {
  i128 base, outer, inner;
  int64_t n_outer, n_inner;
  i128 bytes;
  i128 inner_extent() const { return (n_inner - 1) * inner + bytes; }
  i128 extent() const { return (n_outer - 1) * outer + inner_extent(); }
};
inline Nest nest(const Pieces& p) {
  i128 a = p.rows > 1 ? (i128)p.row : 0, b = p.heads > 1 ? (i128)p.head : 0;
  int64_t na = a ? p.rows : 1, nb = b ? p.heads : 1;  // (a stride of 0 repeats the same pieces)
  if (a < b) {
    std::swap(a, b);
    std::swap(na, nb);
  }
  return {address(p.at), a, b, na, nb, (i128)p.bytes};
}
// Whether a piece of s meets [x, x + bytes).
inline bool meets(const Nest& s, i128 x, i128 bytes) {
  const i128 d = x - s.base, reach = s.inner_extent();
  // outer index o: o * outer - reach < d ... < o * outer + bytes
  int64_t lo = 0, hi = 0;
  if (s.n_outer > 1) {
    const i128 first = d - reach, last = d + bytes;
    lo = first < 0 ? 0 : (int64_t)std::min<i128>(first / s.outer + 1, s.n_outer);
    hi = last <= 0 ? -1 : (int64_t)std::min<i128>((last - 1) / s.outer, s.n_outer - 1);
  }
  for (int64_t o = lo; o <= hi; ++o) {
    const i128 e = d - o * s.outer;  // from the outer piece's begin
    int64_t i = 0;
    if (s.n_inner > 1) i = (int64_t)std::min<i128>(std::max<i128>(e, 0) / s.inner, s.n_inner - 1);
    for (int64_t j = i; j <= i + 1 && j < s.n_inner; ++j)
      if (j * s.inner < e + bytes && e < j * s.inner + s.bytes) return true;
  }
  return false;
}
}  // namespace overlap

// Whether two of a set's own pieces lie on one another.
inline bool meet_themselves(const Pieces& p) {
  if (p.rows == 0 || p.heads == 0) return false;
  if ((p.rows > 1 && p.row < p.bytes) || (p.heads > 1 && p.head < p.bytes)) return true;
  const overlap::Nest s = overlap::nest(p);
  if (s.n_outer == 1 || s.outer >= s.inner_extent()) return false;
  // pieces (0, i) against (o, j): the same as (0, i - j) against (o, 0)
  for (int64_t i = 1; i < s.n_inner; ++i) {
    const overlap::i128 x = i * s.inner;
    for (int64_t o = (int64_t)(x / s.outer); o <= (int64_t)(x / s.outer) + 1 && o < s.n_outer; ++o)
      if (o >= 1 && x < o * s.outer + s.bytes && o * s.outer < x + s.bytes) return true;
  }
  return false;
}

// Whether a piece of a lies on one of b.  Buffers apart, and slices of one
// buffer's rows (or heads), are told at once; anything else piece by piece.
inline bool meet(const Pieces& a, const Pieces& b) {
  if (a.rows == 0 || a.heads == 0 || b.rows == 0 || b.heads == 0) return false;
  const overlap::Nest x = overlap::nest(a), y = overlap::nest(b);
  if (x.base + x.extent() <= y.base || y.base + y.extent() <= x.base) return false;
  if (x.outer == y.outer && x.outer > 0) {
    const overlap::i128 off = ((y.base - x.base) % x.outer + x.outer) % x.outer;
    if (off >= x.inner_extent() && off + y.inner_extent() <= x.outer) return false;
  }
  for (int64_t o = 0; o < x.n_outer; ++o)
    for (int64_t i = 0; i < x.n_inner; ++i)
      if (overlap::meets(y, x.base + o * x.outer + i * x.inner, x.bytes)) return true;
  return false;
}

// The same of two plain ranges.
inline bool meet(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  const overlap::i128 x = overlap::address(a), y = overlap::address(b);
  return a_bytes && b_bytes && x < y + b_bytes && y < x + a_bytes;
}

}  // namespace mit2hip
