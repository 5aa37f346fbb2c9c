// beam_ops.h -- a beam search's step on the GPU (mit2cfm_beam_*): the selection
// over beams and vocabulary, and the reordering of page tables and states.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/mit2cfm.h"

namespace mit2hip {

// Both check their arguments (std::invalid_argument) and enqueue on s without
// waiting or allocating.
void beam_select(const mit2cfm_beam_select& a, hipStream_t s);
void beam_reorder(const mit2cfm_kv_cache& cache, const mit2cfm_beam_reorder& a, hipStream_t s);
// Bytes of beam_select's workspace; 0: an argument out of range.
uint64_t beam_select_workspace(const mit2cfm_beam_select& a);

}  // namespace mit2hip
