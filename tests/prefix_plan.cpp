// The shared-prefix attention's plans (kv_plan.h) over the sizes that its calls accept,
// on the host: every grid can be launched, every key lies in a split, and the splits'
// begins fall on whole tiles and buffers.
#include <cstdio>
#include <random>

#include "kv_plan.h"

using namespace mit2hip;

static int bad = 0, plans = 0, wide = 0, by_xcd = 0, large = 0;

static void check(uint32_t dtype, uint32_t D, uint32_t kv_heads, uint32_t group, uint32_t seqs, uint32_t rows, uint32_t page_rows, uint32_t stride,
                  uint32_t max_length, uint32_t groups, uint32_t max_shared) {
  mit2cfm_kv_cache c{};
  c.dtype = (int32_t)dtype; c.head_dim = D; c.kv_heads = kv_heads; c.page_rows = page_rows; c.table_stride = stride; c.pages = 1;
  mit2cfm_kv_rows r{};
  r.seqs = seqs; r.rows = rows; r.max_length = max_length;
  mit2cfm_kv_prefix x{};
  x.groups = groups; x.max_shared = max_shared;
  const bool f32 = dtype == MIT2CFM_DTYPE_F32;
  const PrefixPlan p = prefix_plan(c, r, kv_heads * group, x);
  const AttendGrid g = attend_grid(p.blocks);
  const int mtile = p.own.form == kWide ? kPrefixRows : 16 * p.own.form;
  // tiles of any division of the rows among n sequences (or groups), the worst: one row each and the rest in one
  auto most_tiles = [&](uint32_t n) {
    const uint64_t fewest = std::min(n, rows);
    return (fewest - 1) * ((group + mtile - 1) / mtile) + ((uint64_t)(rows - fewest + 1) * group + mtile - 1) / mtile;
  };
  auto blocks = [&](const AttendPlan& q) {
    const uint64_t units = (uint64_t)kv_heads * q.splits;
    return q.tiles * (q.by_xcd ? (units + 7) / 8 * 8 : units);
  };
  const uint64_t capacity = (uint64_t)stride * page_rows;
  const uint64_t step = p.own.form == kWide ? wide_keys(D, f32) : chunk_step(f32);
  bool ok = p.own.splits >= 1 && p.own.splits <= kMostSplits && p.own.tiles > 0 && (uint64_t)p.own.tiles >= most_tiles(seqs) && p.own.chunk > 0 &&
            p.own.chunk % step == 0 && shared_step(D, f32) % (f32 ? 16 : 32) == 0 && (shared_step(D, f32) & (shared_step(D, f32) - 1)) == 0;
  if (p.own.form == kWide) ok = ok && shared_step(D, f32) % wide_keys(D, f32) == 0;
  uint64_t all = blocks(p.own);
  if (groups) {
    const uint64_t len = std::max<uint64_t>(1, std::min<uint64_t>(max_shared, capacity));
    ok = ok && p.shared.splits >= 1 && p.shared.splits <= kMostSplits && (uint64_t)p.shared.tiles >= most_tiles(groups) && p.shared.form == p.own.form &&
         p.shared.chunk % step == 0 && (uint64_t)p.shared.chunk * p.shared.splits >= len && p.shared_blocks == blocks(p.shared);
    all += blocks(p.shared);
    by_xcd += p.shared.by_xcd;
  } else {
    ok = ok && p.shared.splits == 0 && p.shared_blocks == 0;
  }
  ok = ok && all == p.blocks && p.slots() <= 2 * kMostSplits;
  ok = ok && (uint64_t)g.x * kAttendThreads < (uint64_t(1) << 32) && g.y < 65536 && (uint64_t)g.x * g.y >= p.blocks && (uint64_t)g.x * g.y < (uint64_t(1) << 32);
  if (!ok) {
    std::printf("dtype %u D %u heads %u x %u seqs %u rows %u length %u groups %u shared %u: form %d own %d x %d of %d, shared %d x %d of %d, blocks %u + .. %u\n", dtype, D,
                kv_heads, group, seqs, rows, max_length, groups, max_shared, p.own.form, p.own.tiles, p.own.splits, p.own.chunk, p.shared.tiles, p.shared.splits,
                p.shared.chunk, p.shared_blocks, p.blocks);
    ++bad;
  }
  ++plans;
  wide += p.own.form == kWide;
  by_xcd += p.own.by_xcd;
  large += p.blocks >= (1u << 24);
}

int main() {
  std::mt19937_64 rng(7);
  auto upto = [&](uint64_t most) {  // spread over the logarithm
    const int bits = 64 - __builtin_clzll(most);
    const uint64_t x = rng() >> (64 - 1 - rng() % bits);
    return 1 + (x - 1) % most;
  };
  const uint32_t dims[] = {32, 64, 96, 128, 192, 256};
  for (int t = 0; t < 300000; ++t) {
    const uint32_t kv = (uint32_t)upto(1024), group = (uint32_t)upto(4096 / kv), page = 1u << rng() % 11;
    const uint64_t most = std::min<uint64_t>((1u << 24) - 1, (uint64_t(1) << 28) / (kv * group));
    const uint32_t rows = (uint32_t)(rng() % 4 ? upto(most) : most), seqs = (uint32_t)upto(65535);
    check(rng() % 3, dims[rng() % 6], kv, group, seqs, rows, page, (uint32_t)upto((1u << 30) / page), (uint32_t)(rng() % 9 ? upto(1u << 31) : rng() % 2),
          rng() % 5 ? (uint32_t)upto(65535) : 0, (uint32_t)(rng() % 9 ? upto(0xffffffffu) : rng() % 2));
  }
  std::printf("%d plans, %d wide, %d by XCD, %d of many blocks, %d wrong\n", plans, wide, by_xcd, large, bad);
  return bad || !wide || !by_xcd || !large ? 1 : 0;
}
