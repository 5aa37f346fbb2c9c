// kv_ops.h -- operators over a paged key/value cache (mit2cfm_kv_*): appending
// new rows with their rotation, and the attention of new rows, single tokens,
// chains or trees of drafted tokens, over the cached ones.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/mit2cfm.h"

namespace mit2hip {

// Both check their arguments (std::invalid_argument) and enqueue on s without
// waiting or allocating.
void kv_append(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, const mit2cfm_kv_append& a, hipStream_t s);
void kv_attention(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, const mit2cfm_kv_attention& a,
                  hipStream_t s);
// Bytes of kv_attention's workspace; 0: none needed, or an argument out of range.
uint64_t kv_attention_workspace(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, uint32_t q_heads);

// Whether a cache's sizes, type and pointers are within their ranges (throws
// std::invalid_argument otherwise); bytes of an element.
void check_kv_cache(const mit2cfm_kv_cache& cache);
int kv_elem_bytes(int32_t dtype);

}  // namespace mit2hip
