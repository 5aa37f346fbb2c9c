// kv_prefix.hip -- attention of sequences that share their first rows: its arguments
// and workspace (the kernels: kv_attend.h, kv_prefix.h).
#include "kv_prefix.h"

#include "kv_args.h"

namespace mit2hip {

namespace {
uint64_t workspace_of(const PrefixPlan& plan, const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads) {
  return (uint64_t)r.rows * q_heads * ((uint64_t)plan.slots() * (c.head_dim + 2) + 2) * sizeof(float);
}
}  // namespace

uint64_t kv_prefix_attention_workspace(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads,
                                       const mit2cfm_kv_prefix& x) {
  try {
    check_kv_sizes(c);
    check_kv_rows(r);
  } catch (const std::invalid_argument&) {
    return 0;
  }
  if (r.seqs == 0 || r.rows == 0 || !query_rows_in_range(c, r, q_heads) || x.groups > 65535) return 0;
  return workspace_of(prefix_plan(c, r, q_heads, x), c, r, q_heads);
}

void kv_prefix_attention(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, const mit2cfm_kv_attention& p,
                         const mit2cfm_kv_prefix& x, hipStream_t s) {
  PrefixArgs a{};
  need(x.groups <= 65535, "groups must be <= 65535");
  need(aligned(x.group, 4) && aligned(x.shared, 4) && aligned(x.lse, 4), "group, shared and lse must be 4-byte aligned");
  if (!attention_args(c, r, p, a)) return;
  need(x.groups == 0 || (x.group && x.shared), "group and shared must not be NULL");
  if (x.lse) {
    const size_t e = (size_t)kv_elem_bytes(c.dtype);
    const Pieces lse = whole(x.lse, (uint64_t)r.rows * p.q_heads * 4);
    need(!meet(pieces(p.q, p.q_row, p.q_head, r.rows, p.q_heads, c.head_dim, e), lse) &&
             !meet(pieces(p.out, p.out_row, p.out_head, r.rows, p.q_heads, c.head_dim, e), lse),
         "lse overlaps q or out");
  }
  const PrefixPlan plan = prefix_plan(c, r, p.q_heads, x);
  need(p.workspace && p.workspace_bytes >= workspace_of(plan, c, r, p.q_heads), "workspace is NULL or too small");
  a.bounds = x.group;
  a.shared = x.shared;
  a.groups = (int)x.groups;
  const int D = (int)c.head_dim;
  if (c.dtype == MIT2CFM_DTYPE_F32)
    launch_prefix_f32(a, plan, D, p.workspace, x.lse, s);
  else if (c.dtype == MIT2CFM_DTYPE_F16)
    launch_prefix_f16(a, plan, D, p.workspace, x.lse, s);
  else
    launch_prefix_bf16(a, plan, D, p.workspace, x.lse, s);
}

}  // namespace mit2hip
