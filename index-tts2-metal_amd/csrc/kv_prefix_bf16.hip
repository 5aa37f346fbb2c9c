// kv_prefix_bf16.hip -- the shared-prefix attention's kernels for bf16 caches (kv_prefix.h).
#define KV_ATTEND_KERNELS
#include "kv_prefix.h"

namespace mit2hip {

void launch_prefix_bf16(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s) {
  launch_prefix_dim<bf16_t>(a, plan, D, workspace, lse, s);
}

}  // namespace mit2hip
