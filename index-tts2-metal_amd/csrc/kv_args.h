// kv_args.h -- what the paged-cache operators (kv_*.hip) do with their arguments on
// the host: refusals, the kernels' views of a cache and its rows, launch errors.
#pragma once

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "engine.h"
#include "kv_attend.h"
#include "kv_ops.h"
#include "kv_view.h"
#include "overlap.h"

namespace mit2hip {

inline void need(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}
inline void kv_launched(hipError_t e) {
  if (e != hipSuccess) throw HipError(std::string("kv operator launch: ") + hipGetErrorString(e));
}
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline CacheView view(const mit2cfm_kv_cache& c) {
  return {static_cast<char*>(c.k), static_cast<char*>(c.v), c.table, (int)c.pages,
          __builtin_ctz(c.page_rows), (int)c.kv_heads, (int)c.table_stride};
}
inline RowView view(const mit2cfm_kv_rows& r) { return {r.start, r.length, (int)r.seqs, (int)r.rows}; }

inline void check_kv_rows(const mit2cfm_kv_rows& r) {
  need(r.seqs <= 65535, "seqs must be <= 65535");
  need(r.rows < (1u << 24), "rows must be below 2^24");
  need(r.seqs == 0 || r.rows == 0 || (r.start && r.length), "start and length must not be NULL");
  need(aligned(r.start, 4) && aligned(r.length, 4), "start and length must be 4-byte aligned");
}

// What the attention's plans, and the kernels' 32-bit numbers of query rows, are made for.
inline bool query_rows_in_range(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads) {
  return q_heads >= 1 && q_heads <= 4096 && q_heads % c.kv_heads == 0 && (uint64_t)r.rows * q_heads <= (1u << 28);
}
inline void set_scale(AttendArgs& a, float scale) {
  a.flip = scale < 0.f;
  a.scale2 = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-37f);  // (0: masked scores stay -inf)
}
// A plain range among sets of pieces.
inline Pieces whole(const void* at, uint64_t bytes) { return {at, 0, 0, 1, 1, bytes}; }

// What an append's kernels take (kv_ops.hip, kv_norm.hip).
struct AppendArgs {
  CacheView c;
  RowView r;
  const char *k, *v, *q;
  char* q_out;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head, qo_row, qo_head;
  const int32_t* position;
  int q_heads, rot, interleaved;
  double log2_theta;
};
constexpr int kMaxPairs = 128;  // rotated pairs of a head
// Checks an append's arguments; false: there are no rows.
bool append_args(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, const mit2cfm_kv_append& p, AppendArgs& a);
// Whether rows may be taken 16 bytes (V elements) at a time.
inline bool append_wide(const AppendArgs& a, int V) {
  auto fits = [&](const void* p, int64_t row, int64_t head) { return aligned(p, 16) && row % V == 0 && head % V == 0; };
  return fits(a.k, a.k_row, a.k_head) && fits(a.v, a.v_row, a.v_head) &&
         (!a.q_heads || (fits(a.q, a.q_row, a.q_head) && fits(a.q_out, a.qo_row, a.qo_head))) &&
         (a.interleaved || a.rot % (2 * V) == 0);
}

// Checks an attention's arguments but for its workspace's size; false: there are no rows.
bool attention_args(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, const mit2cfm_kv_attention& p, AttendArgs& a);

// N elements that are read or written at once.
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

}  // namespace mit2hip
