// kv_prefix_f16.hip -- the shared-prefix attention's kernels for f16 caches (kv_prefix.h).
#define KV_ATTEND_KERNELS
#include "kv_prefix.h"

namespace mit2hip {

void launch_prefix_f16(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s) {
  launch_prefix_dim<half_t>(a, plan, D, workspace, lse, s);
}

}  // namespace mit2hip
