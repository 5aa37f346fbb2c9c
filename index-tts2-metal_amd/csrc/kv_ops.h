// kv_ops.h -- operators over a paged key/value cache (mit2cfm_kv_*): appending
// new rows with their rotation, and the attention of new rows, single tokens,
// chains or trees of drafted tokens, over the cached ones.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/mit2cfm.h"

namespace mit2hip {

// All check their arguments (std::invalid_argument) and enqueue on s without
// waiting or allocating.
void kv_append(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, const mit2cfm_kv_append& a, hipStream_t s);
// The same with normalised queries and keys (kv_norm.hip).
void kv_norm_append(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, const mit2cfm_kv_append& a,
                    const mit2cfm_kv_norm& n, hipStream_t s);
void kv_attention(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, const mit2cfm_kv_attention& a,
                  hipStream_t s);
// Attention of sequences that share their first rows (kv_prefix.hip), and its
// workspace's bytes, 0: an argument out of range.
void kv_prefix_attention(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, const mit2cfm_kv_attention& a,
                         const mit2cfm_kv_prefix& x, hipStream_t s);
uint64_t kv_prefix_attention_workspace(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, uint32_t q_heads,
                                       const mit2cfm_kv_prefix& x);
// Adds up the attention weight that cached rows get (kv_weigh.hip).
void kv_weigh(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, const mit2cfm_kv_weigh& w, hipStream_t s);
// Bytes of kv_attention's workspace; 0: none needed, or an argument out of range.
uint64_t kv_attention_workspace(const mit2cfm_kv_cache& cache, const mit2cfm_kv_rows& rows, uint32_t q_heads);

// Rows of least weight leave the caches of all layers (kv_evict.hip); the bytes of its
// workspace, 0: an argument out of range.
void kv_evict(const mit2cfm_kv_cache& cache, const mit2cfm_kv_evict& e, hipStream_t s);
uint64_t kv_evict_workspace(const mit2cfm_kv_cache& cache, const mit2cfm_kv_evict& e);

// Whether a cache's sizes and type, and its pointers too, are within their ranges
// (throw std::invalid_argument otherwise); bytes of an element.
void check_kv_sizes(const mit2cfm_kv_cache& c);
void check_kv_cache(const mit2cfm_kv_cache& cache);
int kv_elem_bytes(int32_t dtype);

}  // namespace mit2hip
