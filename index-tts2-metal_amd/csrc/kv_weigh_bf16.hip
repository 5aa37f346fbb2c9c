// kv_weigh_bf16.hip -- the added-up attention weights' kernels for bf16 caches (kv_weigh.h).
#define KV_ATTEND_KERNELS
#include "kv_weigh.h"

namespace mit2hip {

void launch_weigh_bf16(const WeighArgs& w, const WeighPlan& plan, int D, hipStream_t s) {
  launch_weigh_dim<bf16_t>(w, plan, D, s);
}

}  // namespace mit2hip
