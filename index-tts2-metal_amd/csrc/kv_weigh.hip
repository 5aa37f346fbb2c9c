// kv_weigh.hip -- adding up the attention weight that cached rows get: its arguments
// (the kernels: kv_weigh.h; how their launch is laid out: kv_plan.h).
#include "kv_weigh.h"

#include <algorithm>
#include <cmath>

#include "kv_args.h"

namespace mit2hip {

void kv_weigh(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, const mit2cfm_kv_weigh& p, hipStream_t s) {
  check_kv_cache(c);
  check_kv_rows(r);
  need(query_rows_in_range(c, r, p.q_heads), "q_heads must be a multiple of kv_heads, <= 4096, rows * q_heads <= 2^28");
  need(std::isfinite(p.scale), "scale must be finite");
  need(std::isfinite(p.decay), "decay must be finite");
  need(p.mask == nullptr || p.mask_words >= 1, "mask_words must be >= 1 with a mask");
  need(p.mask_words < (1u << 24), "mask_words must be below 2^24");
  need(p.weight_stride >= 1 && p.weight_stride <= (1u << 30), "weight_stride must be in [1, 2^30]");
  need(aligned(p.mask, 4) && aligned(p.lse, 4) && aligned(p.weights, 4) && aligned(p.weights_out, 4) && aligned(p.position, 4) &&
           aligned(p.born, 4),
       "mask, lse, weights, weights_out, position and born must be 4-byte aligned");
  if (r.seqs == 0 || r.rows == 0) return;
  need(p.q && p.lse && p.weights && p.weights_out, "q, lse, weights and weights_out must not be NULL");
  const size_t e = (size_t)kv_elem_bytes(c.dtype);
  need(aligned(p.q, e), "q must be aligned to its type");
  const uint64_t bytes = (uint64_t)r.seqs * c.kv_heads * p.weight_stride * 4;
  const uint64_t lse_bytes = (uint64_t)r.rows * p.q_heads * 4, mask_bytes = p.mask ? (uint64_t)r.rows * p.mask_words * 4 : 0;
  const Pieces q = pieces(p.q, p.q_row, p.q_head, r.rows, p.q_heads, c.head_dim, e);
  need(p.weights == p.weights_out || !meet(p.weights, bytes, p.weights_out, bytes), "weights_out overlaps weights");
  need(!meet(q, whole(p.weights_out, bytes)) && !meet(p.lse, lse_bytes, p.weights_out, bytes) &&
           !meet(p.mask, mask_bytes, p.weights_out, bytes),
       "weights_out overlaps q, lse or mask");
  if (p.born) {
    need(!meet(p.born, bytes, p.weights, bytes) && !meet(p.born, bytes, p.weights_out, bytes) && !meet(q, whole(p.born, bytes)) &&
             !meet(p.lse, lse_bytes, p.born, bytes) && !meet(p.mask, mask_bytes, p.born, bytes) &&
             !(p.position && meet(p.position, (uint64_t)r.rows * 4, p.born, bytes)),
         "born overlaps another buffer");
  }
  WeighArgs w{};
  AttendArgs& a = w.a;
  a.c = view(c);
  a.r = view(r);
  a.q = static_cast<const char*>(p.q);
  a.q_row = (int64_t)p.q_row; a.q_head = (int64_t)p.q_head;
  a.mask = p.mask;
  a.mask_words = p.mask ? (int)p.mask_words : 0;
  a.q_heads = (int)p.q_heads;
  a.group = (int)(p.q_heads / c.kv_heads);
  w.c2 = p.scale * 1.4426950408889634f;
  a.q_wide = aligned(p.q, 16) && p.q_row % 8 == 0 && p.q_head % 8 == 0;
  w.lse = p.lse;
  w.weights = p.weights;
  w.weights_out = p.weights_out;
  w.stride = p.weight_stride;
  w.decay = p.decay;
  w.last_rows = (int)std::min(p.last_rows, 1u << 24);
  w.position = p.position;
  w.born = p.born;
  const int D = (int)c.head_dim;
  const WeighPlan plan = weigh_plan(c, r, p.q_heads, p.last_rows, p.weight_stride);
  if (c.dtype == MIT2CFM_DTYPE_F32)
    launch_weigh_f32(w, plan, D, s);
  else if (c.dtype == MIT2CFM_DTYPE_F16)
    launch_weigh_f16(w, plan, D, s);
  else
    launch_weigh_bf16(w, plan, D, s);
}

}  // namespace mit2hip
