// kv_plan.h -- how the paged attention's launches are laid out (kv_attend.h), from
// sizes alone (host).
#pragma once

#include <algorithm>
#include <cstdint>

#include "../../include/mit2cfm.h"

namespace mit2hip {

// How a launch is laid out (attend_plan).
struct AttendPlan {
  int form;    // query tiles a wave (1, 2), kWide: the block kernel
  int tiles;   // query tiles of the batch, an upper bound
  int splits;  // of a sequence's keys, at most
  int chunk;   // keys of a split, unless the sequence is longer than splits of them
  int by_xcd;  // blocks of a key head and split on one XCD (see find_part)
};
constexpr int kWide = 0;
constexpr int kAttendWaves = 4, kAttendThreads = kAttendWaves * 64;
// A split of the small tiles is a multiple of this, a tile for each of a block's
// waves; one of the block form has as many keys at least.
constexpr int chunk_step(bool f32) { return f32 ? 64 : 128; }

// Query rows of the block kernel's tile, and the head sizes it is made for.
constexpr int wide_rows(bool f32) { return f32 ? 64 : 128; }
constexpr bool wide_dim(int D) { return D == 64 || D == 128; }

constexpr int kBlocksWanted = 1024;   // four blocks of the small tiles a CU
// Blocks of the wide form that run at once on 256 CUs: two a CU at 128 elements of
// 16 bits (by registers), else three (by LDS).
constexpr int wide_places(int D, bool f32) { return 256 * (D == 128 && !f32 ? 2 : 3); }
// Keys of one of its buffers; a split's are a multiple of this.
constexpr int wide_keys(int D, bool f32) { return 8192 / (D * (f32 ? 4 : 2)); }
constexpr int kMostSplits = 128;

// Splits of `len` keys for `blocks` wide blocks: those with which the rounds that the
// blocks run in, times a block's keys, are least.  A block's begin and end (the
// ring's fill, the last buffers' waits) count as four buffers, a join as four more.
// (A fixed 640 for 512 places went in two rounds where the tiles' number is exact:
// 63 rows of 32 heads on 8 of 128 f16 over 4099, 32768, 65536 keys took 41, 79, 128 us
// so, 35, 67, 107 now; a prompt of 2047 in bf16 105, now 75; 30 sequences of 40 rows over
// 2000 keys 108, now 92.  Of 8 ragged ones, whose shorter leave places free, it was
// faster: 55, now 59.)
inline uint64_t wide_splits(uint64_t blocks, uint64_t len, uint64_t places, uint64_t step, uint64_t most) {
  uint64_t best = 1, least = ~uint64_t(0);
  const uint64_t first = (blocks + places - 1) / places;  // rounds without a split
  for (uint64_t r = first; r < first + 3; ++r) {
    const uint64_t s = std::min(std::max<uint64_t>(1, r * places / blocks), most);
    const uint64_t keys = ((len + s - 1) / s + step - 1) / step * step;
    const uint64_t cost = (blocks * s + places - 1) / places * (keys + 4 * step) + (s > 1 ? 4 * step : 0);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

inline AttendPlan attend_plan(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads) {
  const int group = (int)(q_heads / c.kv_heads), D = (int)c.head_dim;
  const bool f32 = c.dtype == MIT2CFM_DTYPE_F32;
  // Query rows of a tile follow the average sequence's.  Of 8 heads of 128 f16 in 8
  // sequences of 4000 keys, 16 rows take 32, 43, 28 us with one tile, two, and the block
  // kernel, 32 rows 49, 44, 32, 64 rows 82, 65, 37; 24 rows over 131001 bf16 keys 154,
  // 119, 139; and one row of each of 64 sequences, the decoding step, 187, -, 193.
  // Of heads of 64, and of fp32, the block kernel gains later: 20 heads of 64 f16 take 56,
  // 43, 46 us at 32 rows, 77, 61, 50 at 48; fp32 111, 79, 111 and 164, 142, 146 (in 2
  // sequences 34, 28, 35 and 47, 44, 39).  Four tiles a wave were slower than two.
  const uint64_t m = (uint64_t)r.rows * group / r.seqs;
  AttendPlan p;
  p.form = wide_dim(D) && m > (D == 128 && !f32 ? 16 : 32) ? kWide : m <= 16 ? 1 : 2;
  const int mtile = p.form == kWide ? wide_rows(f32) : 16 * p.form;
  // sum over the sequences of ceil(rows * group / mtile): at most ...
  const uint64_t by_fill = ((uint64_t)r.rows * group + (uint64_t)std::min(r.seqs, r.rows) * (mtile - 1)) / mtile;
  const uint64_t by_row = (uint64_t)r.rows * ((group + mtile - 1) / mtile);
  p.tiles = (int)std::min(by_fill, by_row);
  const uint64_t len = std::max<uint64_t>(1, std::min<uint64_t>(r.max_length, (uint64_t)c.table_stride * c.page_rows));
  const uint64_t step = p.form == kWide ? wide_keys(D, f32) : chunk_step(f32);
  const uint64_t most = std::min<uint64_t>((len + chunk_step(f32) - 1) / chunk_step(f32), kMostSplits);
  uint64_t splits;
  if (p.form == kWide) {
    // (as if the rows were spread evenly; of one sequence the number is exact)
    const uint64_t each = ((uint64_t)r.rows + r.seqs - 1) / r.seqs;
    const uint64_t even = std::min<uint64_t>(p.tiles, r.seqs * ((each * group + mtile - 1) / mtile));
    splits = wide_splits(even * c.kv_heads, len, wide_places(D, f32), step, most);
  } else {
    const uint64_t blocks = (uint64_t)p.tiles * c.kv_heads;
    splits = std::min<uint64_t>(most, (kBlocksWanted + blocks - 1) / blocks);
  }
  p.chunk = (int)(((len + splits - 1) / splits + step - 1) / step * step);
  p.splits = (int)((len + p.chunk - 1) / p.chunk);
  const uint64_t units = (uint64_t)c.kv_heads * p.splits;
  // (all in x then, which holds fewer than 2^32 threads)
  p.by_xcd = p.form == kWide && (units % 8 == 0 || units >= 32) &&
             (units + 7) / 8 * 8 * p.tiles < (uint64_t(1) << 32) / kAttendThreads;
  return p;
}

// The grid of a plan's blocks.
struct AttendGrid {
  uint32_t x, y;
};
inline AttendGrid attend_grid(const AttendPlan& plan, int kv_heads) {
  const uint32_t units = (uint32_t)kv_heads * plan.splits, tiles = (uint32_t)plan.tiles;
  return plan.by_xcd ? AttendGrid{8 * ((units + 7) / 8) * tiles, 1} : AttendGrid{tiles, units};
}

}  // namespace mit2hip
