// kv_attend_f16.hip -- the paged attention's kernels for f16 caches (kv_attend.h).
#define KV_ATTEND_KERNELS
#include "kv_attend.h"

namespace mit2hip {

void launch_attend_f16(const AttendArgs& a, const AttendPlan& plan, int D, void* workspace, hipStream_t s) {
  launch_attend_dim<half_t>(a, plan, D, workspace, s);
}

}  // namespace mit2hip
