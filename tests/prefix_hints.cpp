// The shared-prefix attention's plans (kv_plan.h) at the largest lengths that can be said:
// laid out for what the table holds, as lengths just past that are.
#include <cstdio>

#include "kv_plan.h"

using namespace mit2hip;

int main() {
  int bad = 0, plans = 0;
  for (uint32_t dtype : {MIT2CFM_DTYPE_F32, MIT2CFM_DTYPE_F16, MIT2CFM_DTYPE_BF16})
    for (uint32_t D : {32u, 64u, 96u, 128u, 192u, 256u})
      for (uint32_t rows : {1u, 9u, 300u})
        for (uint32_t shared : {0u, 1u, 20u, 63u, 64u, 500u, 100000u, 0xffffffffu})
          for (uint32_t length : {0xffffffffu, 0xfffffffeu, 0xffffffc0u, 0x80000000u}) {
            mit2cfm_kv_cache c{};
            c.dtype = (int32_t)dtype; c.head_dim = D; c.kv_heads = 4; c.page_rows = 64; c.table_stride = 2048; c.pages = 1;
            mit2cfm_kv_rows r{};
            r.seqs = 1; r.rows = rows; r.max_length = length;
            mit2cfm_kv_prefix x{};
            x.groups = 1; x.max_shared = shared;
            const PrefixPlan p = prefix_plan(c, r, 8, x);
            // the same, said as little more than the table has (own rows past the shared ones)
            r.max_length = length > shared ? std::min(length, std::min(shared, 1u << 30) + (1u << 18)) : length;
            const PrefixPlan q = prefix_plan(c, r, 8, x);
            ++plans;
            if (p.own.splits != q.own.splits || p.own.chunk != q.own.chunk || p.shared.splits != q.shared.splits || p.blocks != q.blocks) {
              std::printf("dtype %u D %u rows %u shared %u length %u: %d x %d, said less %d x %d\n", dtype, D, rows, shared, length, p.own.splits, p.own.chunk, q.own.splits,
                          q.own.chunk);
              ++bad;
            }
          }
  std::printf("%d plans, %d wrong\n", plans, bad);
  return bad != 0;
}
