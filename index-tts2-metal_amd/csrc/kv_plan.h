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

// The same where prefixes are shared: three blocks fit on a CU (64 tokens on one prefix of
// 8191 bf16 rows 48 us, with 128 rows and two blocks 70, and parts of twice the bytes).
constexpr int kPrefixRows = 64;
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

// The form for the rows of a batch.
inline int attend_form(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads) {
  const int D = (int)c.head_dim;
  const bool f32 = c.dtype == MIT2CFM_DTYPE_F32;
  // Query rows of a tile follow the average sequence's.  Of 8 heads of 128 f16 in 8
  // sequences of 4000 keys, 16 rows take 32, 43, 28 us with one tile, two, and the block
  // kernel, 32 rows 49, 44, 32, 64 rows 82, 65, 37; 24 rows over 131001 bf16 keys 154,
  // 119, 139; and one row of each of 64 sequences, the decoding step, 187, -, 193.
  // Of heads of 64, and of fp32, the block kernel gains later: 20 heads of 64 f16 take 56,
  // 43, 46 us at 32 rows, 77, 61, 50 at 48; fp32 111, 79, 111 and 164, 142, 146 (in 2
  // sequences 34, 28, 35 and 47, 44, 39).  Four tiles a wave were slower than two.
  const uint64_t m = (uint64_t)r.rows * (q_heads / c.kv_heads) / r.seqs;
  return wide_dim(D) && m > (D == 128 && !f32 ? 16 : 32) ? kWide : m <= 16 ? 1 : 2;
}
// Query tiles of a form, for any division of the rows among the sequences.
inline int attend_tiles(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads, int mtile) {
  const int group = (int)(q_heads / c.kv_heads);
  // sum over the sequences of ceil(rows * group / mtile): at most ...
  const uint64_t by_fill = ((uint64_t)r.rows * group + (uint64_t)std::min(r.seqs, r.rows) * (mtile - 1)) / mtile;
  const uint64_t by_row = (uint64_t)r.rows * ((group + mtile - 1) / mtile);
  return (int)std::min(by_fill, by_row);
}
// Keys that a launch is laid out for.
inline uint64_t attend_length(const mit2cfm_kv_cache& c, uint64_t hint) {
  return std::max<uint64_t>(1, std::min<uint64_t>(hint, (uint64_t)c.table_stride * c.page_rows));
}
// Whether blocks go by XCDs (all in x then, which holds fewer than 2^32 threads).
inline bool attend_by_xcd(const AttendPlan& p, uint32_t kv_heads) {
  const uint64_t units = (uint64_t)kv_heads * p.splits;
  return p.form == kWide && (units % 8 == 0 || units >= 32) &&
         (units + 7) / 8 * 8 * p.tiles < (uint64_t(1) << 32) / kAttendThreads;
}

inline AttendPlan attend_plan(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads) {
  const int group = (int)(q_heads / c.kv_heads), D = (int)c.head_dim;
  const bool f32 = c.dtype == MIT2CFM_DTYPE_F32;
  AttendPlan p;
  p.form = attend_form(c, r, q_heads);
  const int mtile = p.form == kWide ? wide_rows(f32) : 16 * p.form;
  p.tiles = attend_tiles(c, r, q_heads, mtile);
  const uint64_t len = attend_length(c, r.max_length);
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
  p.by_xcd = attend_by_xcd(p, c.kv_heads);
  return p;
}

// The two halves of an attention of shared prefixes, one launch: the same form for
// both, the one that the more rows a tile ask for, and splits of about as many keys.
struct PrefixPlan {
  AttendPlan shared, own;  // shared.splits 0: nothing is shared
  uint32_t shared_blocks, blocks;
  int slots() const { return shared.splits + own.splits; }
};
// Shared rows are taken in runs of this: a tile's keys, a buffer's of the block form.
constexpr int shared_step(int D, bool f32) {
  return std::max(f32 ? 16 : 32, wide_dim(D) ? wide_keys(D, f32) : 0);
}
inline PrefixPlan prefix_plan(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads, const mit2cfm_kv_prefix& x) {
  const int D = (int)c.head_dim;
  const bool f32 = c.dtype == MIT2CFM_DTYPE_F32, shares = x.groups > 0;
  mit2cfm_kv_rows some = r;
  some.seqs = std::max(x.groups, 1u);
  PrefixPlan p{};
  const int form = attend_form(c, r, q_heads), wider = shares ? attend_form(c, some, q_heads) : form;
  p.shared.form = p.own.form = form == kWide || wider == kWide ? kWide : std::max(form, wider);
  const int mtile = p.own.form == kWide ? kPrefixRows : 16 * p.own.form;
  p.shared.tiles = shares ? attend_tiles(c, some, q_heads, mtile) : 0;
  p.own.tiles = attend_tiles(c, r, q_heads, mtile);
  const uint64_t shared_len = shares ? attend_length(c, x.max_shared) : 0;
  const uint64_t past = r.max_length > x.max_shared ? (uint64_t)r.max_length - x.max_shared + shared_step(D, f32) - 1 : 1;
  const uint64_t own_len = attend_length(c, shares ? past : r.max_length);
  const uint64_t step = p.own.form == kWide ? wide_keys(D, f32) : chunk_step(f32), longest = std::max(shared_len, own_len);
  auto splits = [](uint64_t len, uint64_t chunk) { return (len + chunk - 1) / chunk; };
  // What a chunk costs, in a block's steps on a CU (0.5 us each where its places are
  // taken, half as much again for a block alone): the shared rows' blocks lie side by side
  // on the CUs, each as long as the longest, the others fill in; a block's begin and end
  // count as six steps, and its parts are written and read again at 4 TB/s.  (As if the
  // rows were spread evenly.)
  auto even = [&](uint32_t seqs) {
    const uint64_t each = ((uint64_t)r.rows + seqs - 1) / seqs;
    return seqs * ((each * (q_heads / c.kv_heads) + mtile - 1) / mtile) * c.kv_heads;
  };
  const uint64_t shared_units = shares ? std::min<uint64_t>(even(some.seqs), (uint64_t)p.shared.tiles * c.kv_heads) : 0;
  const uint64_t own_units = std::min<uint64_t>(even(r.seqs), (uint64_t)p.own.tiles * c.kv_heads);
  const double parts_step = (double)r.rows * q_heads * (D + 2) * 8.0 / 4e6 / 0.5;
  auto cost = [&](uint64_t chunk) {
    const uint64_t ns = splits(shared_len, chunk), no = splits(own_len, chunk);
    const uint64_t bs = shared_units * ns, bo = own_units * no;
    const double ls = (double)std::min(chunk, shared_len) / step + 6.0, lo = (double)std::min(chunk, own_len) / step + 6.0;
    const double load = bs ? (bs + 255) / 256 * ls + bo * lo / 256.0 : (bo + 255) / 256 * lo;
    return std::max(load, 1.5 * std::max(bs ? ls : 0.0, lo)) + parts_step * (ns + no);
  };
  uint64_t chunk = 0;
  double least = 0.0;
  auto consider = [&](uint64_t len, uint64_t units) {  // with 1 to 4 blocks a CU of them, and no splits
    for (uint64_t k = 0; k <= 4 && len; ++k) {
      const uint64_t n = std::min<uint64_t>(std::max<uint64_t>(1, k * 256 / units), kMostSplits);
      if (k && n == 1) continue;
      uint64_t x = std::max((len + n - 1) / n, (longest + kMostSplits - 1) / kMostSplits);
      x = (x + step - 1) / step * step;
      const double y = cost(x);
      if (chunk == 0 || y < least) {
        chunk = x;
        least = y;
      }
    }
  };
  consider(shared_len, shared_units);
  consider(own_len, own_units);
  p.shared.chunk = p.own.chunk = (int)chunk;
  p.shared.splits = (int)splits(shared_len, p.shared.chunk);
  p.own.splits = (int)splits(own_len, p.own.chunk);
  p.shared.by_xcd = shares && attend_by_xcd(p.shared, c.kv_heads);
  p.own.by_xcd = attend_by_xcd(p.own, c.kv_heads);
  auto count = [&](const AttendPlan& q) {
    const uint64_t units = (uint64_t)c.kv_heads * q.splits;
    return (uint32_t)(q.tiles * (q.by_xcd ? (units + 7) / 8 * 8 : units));
  };
  p.shared_blocks = shares ? count(p.shared) : 0;
  p.blocks = p.shared_blocks + count(p.own);
  return p;
}

// How the attention weights' launch is laid out (weigh_plan).
struct WeighPlan {
  int by_query;     // a block's waves share their keys and divide the queries
  uint32_t blocks;  // of a sequence and key head
  int by_xcd;       // those on one XCD, whose L2 then has their queries
};
// 16-key tiles of a wave: up to 64 keys, 16 KB of them.
constexpr int weigh_tiles(int D, int bytes) {
  return D * bytes <= 256 ? 4 : D * bytes <= 512 ? 2 : 1;
}
inline WeighPlan weigh_plan(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads, uint32_t last_rows, uint32_t weight_stride) {
  const uint64_t group = q_heads / c.kv_heads, lines = (uint64_t)r.seqs * c.kv_heads;
  const uint64_t len = std::min<uint64_t>({r.max_length, (uint64_t)c.table_stride * c.page_rows, weight_stride});
  const uint64_t wave_keys = 16 * weigh_tiles((int)c.head_dim, c.dtype == MIT2CFM_DTYPE_F32 ? 4 : 2);
  const uint64_t all_blocks = lines * ((len + 4 * wave_keys - 1) / (4 * wave_keys));
  // Waves that divide the queries make four times the blocks, and each loads all of its
  // block's keys: worth it while the blocks of waves with keys of their own do not fill
  // the chip, or where the queries take longer than that.  2047 f16 keys of 128, 8 key
  // heads, 4 query heads each, prompts of as many rows, us with keys of their own / queries
  // divided:
  //              16 rows      64 rows      256 rows     1029 rows
  //   1 prompt   10.0 / 9.0   24.9 / 13.1  54.2 / 21.0  225 / 52
  //   4 prompts  10.2 / 19.7  25.7 / 27.2  66.2 / 44.6  236 / 107
  //   16         25.7 / 56.5  60.4 / 74.1  139 / 129    496 / 319
  const uint64_t each = last_rows ? std::min<uint64_t>(r.rows, (uint64_t)r.seqs * last_rows) : r.rows;
  const uint64_t tiles = each * group / r.seqs / 16;  // of queries, on average
  WeighPlan plan;
  plan.by_query = tiles > std::clamp<uint64_t>(all_blocks / 16, 2, 64);
  const uint64_t keys = wave_keys * (plan.by_query ? 1 : kAttendWaves);
  // With keys of their own, no more blocks than 8 a CU, each then has several chunks: 64
  // sequences of up to 8191 keys 164 us (4 a CU 172, 16 a CU 169, one for each chunk 213).
  const uint64_t most = plan.by_query ? 1u << 20 : std::max<uint64_t>(1, 2048 / lines);
  plan.blocks = (uint32_t)std::clamp<uint64_t>((len + keys - 1) / keys, 1, most);
  // A line's blocks on one XCD, whose L2 has their queries: 4 ragged prompts of 1029 rows
  // 65 us (in launch order 94), 16 of 64 rows 56 (66).
  plan.by_xcd = plan.by_query && (lines % 8 == 0 || lines >= 32) && (lines + 7) * plan.blocks < (1u << 23);
  return plan;
}
// Its blocks in x (y and z: key heads and sequences, unless they go by XCDs).
inline uint32_t weigh_grid(const WeighPlan& plan, uint64_t lines) {
  return plan.by_xcd ? (uint32_t)(8 * ((lines + 7) / 8) * plan.blocks) : plan.blocks;
}

// The grid of a plan's blocks.
struct AttendGrid {
  uint32_t x, y;
};
inline AttendGrid attend_grid(uint32_t blocks) {  // of numbered blocks
  const uint32_t x = std::min(blocks, 1u << 22);
  return {x, (blocks + x - 1) / x};
}
inline AttendGrid attend_grid(const AttendPlan& plan, int kv_heads) {
  const uint32_t units = (uint32_t)kv_heads * plan.splits, tiles = (uint32_t)plan.tiles;
  return plan.by_xcd ? AttendGrid{8 * ((units + 7) / 8) * tiles, 1} : AttendGrid{tiles, units};
}

}  // namespace mit2hip
