// The attention weights' plans (kv_plan.h), on the host: over the sizes that its calls
// accept every grid can be launched; and the form of given sizes, a line each of
// "dtype dim kv_heads group seqs rows max_length page_rows table_stride last_rows weight_stride".
#include <cstdio>
#include <random>

#include "kv_plan.h"

using namespace mit2hip;

struct Sizes {
  uint32_t dtype, dim, kv, group, seqs, rows, max_length, page, table, last, stride;
  WeighPlan plan() const {
    mit2cfm_kv_cache c{};
    c.dtype = (int32_t)dtype; c.head_dim = dim; c.kv_heads = kv; c.page_rows = page; c.table_stride = table; c.pages = 1;
    mit2cfm_kv_rows r{};
    r.seqs = seqs; r.rows = rows; r.max_length = max_length;
    return weigh_plan(c, r, kv * group, last, stride);
  }
};

int main(int argc, char**) {
  if (argc > 1) {
    Sizes z;
    while (std::scanf("%u %u %u %u %u %u %u %u %u %u %u", &z.dtype, &z.dim, &z.kv, &z.group, &z.seqs, &z.rows, &z.max_length, &z.page, &z.table, &z.last, &z.stride) == 11) {
      const WeighPlan p = z.plan();
      std::printf("%d %u %d\n", p.by_query, p.blocks, p.by_xcd);
    }
    return 0;
  }
  std::mt19937_64 rng(7);
  auto upto = [&](uint64_t most) {  // spread over the logarithm
    const int bits = 64 - __builtin_clzll(most);
    const uint64_t x = rng() >> (64 - 1 - rng() % bits);
    return 1 + (x - 1) % most;
  };
  const uint32_t dims[] = {32, 64, 96, 128, 192, 256};
  int bad = 0, forms[2] = {}, by_xcd = 0;
  for (int t = 0; t < 300000; ++t) {
    Sizes z{(uint32_t)(rng() % 3), dims[rng() % 6]};
    z.kv = (uint32_t)upto(4096);
    z.group = (uint32_t)upto(4096 / z.kv);
    z.page = 1u << rng() % 11;
    const uint64_t most = std::min<uint64_t>((1u << 24) - 1, (uint64_t(1) << 28) / (z.kv * z.group));
    z.rows = (uint32_t)(rng() % 4 ? upto(most) : most);
    z.seqs = (uint32_t)upto(65535);
    z.table = (uint32_t)upto((1u << 30) / z.page);
    z.max_length = (uint32_t)(rng() % 9 ? upto(0xffffffffu) : rng() % 2);
    z.last = (uint32_t)(rng() % 2 ? 0 : upto(0xffffffffu));
    z.stride = (uint32_t)upto(1u << 30);
    const WeighPlan p = z.plan();
    const uint64_t lines = (uint64_t)z.seqs * z.kv, x = weigh_grid(p, lines);
    bool ok = p.blocks >= 1 && p.blocks <= (1u << 20) && x * kAttendThreads < (uint64_t(1) << 32) && z.kv <= 65535 && z.seqs <= 65535;
    if (p.by_xcd) ok = ok && p.by_query && x == (lines + 7) / 8 * 8 * p.blocks && x / 8 % p.blocks == 0;
    if (!ok) {
      std::printf("dtype %u dim %u heads %u x %u seqs %u rows %u length %u: %d %u %d\n", z.dtype, z.dim, z.kv, z.group, z.seqs, z.rows, z.max_length, p.by_query, p.blocks,
                  p.by_xcd);
      ++bad;
    }
    ++forms[p.by_query];
    by_xcd += p.by_xcd;
  }
  std::printf("%d with keys of their own, %d that divide the queries, %d by XCD, %d wrong\n", forms[0], forms[1], by_xcd, bad);
  return bad || !forms[0] || !forms[1] || !by_xcd ? 1 : 0;
}
