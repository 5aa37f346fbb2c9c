// The paged attention's plans (kv_plan.h) over the sizes that its calls accept, on the
// host: every grid can be launched, and every key of a sequence lies in a split.
#include <cstdio>
#include <random>

#include "kv_plan.h"

using namespace mit2hip;

static int bad = 0, plans = 0, wide = 0, by_xcd = 0, large = 0;

static void check(uint32_t dtype, uint32_t D, uint32_t kv_heads, uint32_t group, uint32_t seqs, uint32_t rows, uint32_t page_rows, uint32_t stride,
                  uint32_t max_length) {
  mit2cfm_kv_cache c{};
  c.dtype = (int32_t)dtype; c.head_dim = D; c.kv_heads = kv_heads; c.page_rows = page_rows; c.table_stride = stride; c.pages = 1;
  mit2cfm_kv_rows r{};
  r.seqs = seqs; r.rows = rows; r.max_length = max_length;
  const AttendPlan p = attend_plan(c, r, kv_heads * group);
  const AttendGrid g = attend_grid(p, (int)kv_heads);
  const int mtile = p.form == kWide ? wide_rows(dtype == MIT2CFM_DTYPE_F32) : 16 * p.form;
  const uint64_t len = std::max<uint64_t>(1, std::min<uint64_t>(max_length, (uint64_t)stride * page_rows));
  // tiles of any division of the rows among the sequences, the worst: one row each and the rest in one
  const uint64_t fewest = std::min(seqs, rows);
  const uint64_t tiles = (fewest - 1) * ((group + mtile - 1) / mtile) + ((uint64_t)(rows - fewest + 1) * group + mtile - 1) / mtile;
  const uint64_t units = (uint64_t)kv_heads * p.splits;
  bool ok = p.tiles > 0 && (uint64_t)p.tiles >= tiles && p.splits >= 1 && p.splits <= kMostSplits && p.chunk > 0 &&
            (uint64_t)p.chunk * p.splits >= len && (uint64_t)p.chunk * (p.splits - 1) < len;
  ok = ok && (uint64_t)g.x * kAttendThreads < (uint64_t(1) << 32) && g.y < 65536 && (uint64_t)g.x * g.y >= (uint64_t)p.tiles * units;
  if (p.by_xcd) ok = ok && p.form == kWide && g.y == 1 && g.x == (units + 7) / 8 * 8 * p.tiles;
  if (!ok) {
    std::printf("dtype %u D %u heads %u x %u seqs %u rows %u length %u: form %d tiles %d splits %d chunk %d xcd %d grid %u %u\n", dtype, D, kv_heads,
                group, seqs, rows, max_length, p.form, p.tiles, p.splits, p.chunk, p.by_xcd, g.x, g.y);
    ++bad;
  }
  ++plans;
  wide += p.form == kWide;
  by_xcd += p.by_xcd;
  large += (uint64_t)p.tiles * units >= (uint64_t(1) << 24);
}

// One sequence's blocks, whose number is exact: how many rounds they run in, times a
// block's keys, against the keys and tiles spread evenly over the chip.
static void even(uint32_t dtype, uint32_t D, uint32_t kv_heads, uint32_t group, uint32_t rows, uint32_t length, uint64_t at_once, double most) {
  mit2cfm_kv_cache c{};
  c.dtype = (int32_t)dtype; c.head_dim = D; c.kv_heads = kv_heads; c.page_rows = 64; c.table_stride = length / 64 + 1; c.pages = 1;
  mit2cfm_kv_rows r{};
  r.seqs = 1; r.rows = rows; r.max_length = length;
  const AttendPlan p = attend_plan(c, r, kv_heads * group);
  const uint64_t mtile = dtype == MIT2CFM_DTYPE_F32 ? 64 : 128, tiles = ((uint64_t)rows * group + mtile - 1) / mtile;
  const uint64_t blocks = tiles * kv_heads * p.splits, rounds = (blocks + at_once - 1) / at_once;
  const double share = (double)tiles * kv_heads * length / at_once, longest = (double)rounds * p.chunk;
  if (p.form != kWide || longest > most * share) {
    std::printf("dtype %u D %u heads %u x %u rows %u length %u: %lu blocks of %d keys, %.2f of an even share\n", dtype, D, kv_heads, group, rows, length,
                (unsigned long)blocks, p.chunk, longest / share);
    ++bad;
  }
}

int main() {
  // long contexts of one sequence: within a tenth of an even share (two blocks of 128 elements of 16 bits a CU at once, else three)
  even(MIT2CFM_DTYPE_F16, 128, 8, 4, 63, 32768, 512, 1.1);
  even(MIT2CFM_DTYPE_BF16, 128, 8, 4, 63, 65536, 512, 1.1);
  even(MIT2CFM_DTYPE_BF16, 128, 8, 4, 250, 65536, 512, 1.1);
  even(MIT2CFM_DTYPE_F16, 64, 20, 1, 200, 65536, 768, 1.1);
  even(MIT2CFM_DTYPE_F32, 64, 20, 1, 100, 40000, 768, 1.1);
  // as many blocks as the accepted sizes give: over 2^24, which one dimension of 256 threads each cannot hold
  check(MIT2CFM_DTYPE_F16, 128, 1024, 1, 15419, 262144, 16, 64, 1000);
  check(MIT2CFM_DTYPE_BF16, 128, 240, 1, 65535, 17 * 65535, 16, 64, 1000);
  check(MIT2CFM_DTYPE_F32, 64, 512, 1, 15887, 524288, 16, 64, 1);
  const int known = large;
  std::mt19937_64 rng(3);
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
    check(rng() % 3, dims[rng() % 6], kv, group, seqs, rows, page, (uint32_t)upto((1u << 30) / page), (uint32_t)(rng() % 9 ? upto(1u << 31) : rng() % 2));
  }
  std::printf("%d plans, %d wide, %d by XCD, %d of many blocks (%d known), %d wrong\n", plans, wide, by_xcd, large, known, bad);
  return bad || known < 2 || !wide || !by_xcd ? 1 : 0;
}
