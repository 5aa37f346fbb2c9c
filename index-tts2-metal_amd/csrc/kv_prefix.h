// kv_prefix.h -- attention of sequences that share their first rows
// (mit2cfm_kv_prefix_attention): the launches of one element type, instantiated in
// kv_prefix_{f32,f16,bf16}.hip.
#pragma once

#include "kv_attend.h"

namespace mit2hip {

// Launches both halves and their join; throws HipError.  lse may be NULL.
void launch_prefix_f32(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s);
void launch_prefix_f16(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s);
void launch_prefix_bf16(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s);

#if defined(KV_ATTEND_KERNELS)

// Joins the parts of a row and query head: those of the shared rows, then its
// sequence's own.  Lane groups of D/4 take every so manyth part, four elements a lane,
// AHEAD of them at once; WAVES of them for more parts than those.  Its parts' way through
// the cache bounds it: 48 trees of up to 9 rows, 32 heads of 128, 8 us beside the parts' 52.
constexpr int kJoinFew = 16;
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void join_kernel(PrefixArgs a, int shared_splits, Parts part, float* lse) {
  constexpr int L4 = D / 4, G = WAVES * 64 / L4, AHEAD = 8;
  __shared__ floatx4 sO[G][L4];
  __shared__ float sF[2 * kMostSplits], sM[WAVES], sL[WAVES];
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const size_t pair = (size_t)row * a.q_heads + h, at = pair * (shared_splits + a.own.splits);
  const int first = a.r.start[0], last = a.r.start[a.r.seqs];
  const int told = part.n[pair + a.pairs];
  const int shared_told = shared_splits ? part.n[pair] : 0;
  if (row < first || row >= last) return;  // nobody's row
  const int shared = told >> 16 ? min(max(shared_told, 0), shared_splits) : 0;
  const int n = shared + min(told & 0xffff, a.own.splits);
  auto slot = [&](int i) { return at + (i < shared ? i : shared_splits + i - shared); };
  const int g = tid / L4, l4 = tid - g * L4;
  floatx4 x[AHEAD];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) x[u] = reinterpret_cast<const floatx4*>(part.o + slot(max(min(g + u * G, n - 1), 0)) * D)[l4];
  float mm = -INFINITY;
  for (int i = tid; i < n; i += WAVES * 64) mm = fmaxf(mm, part.ml[slot(i)].x);
#pragma unroll
  for (int off = 32; off; off >>= 1) mm = fmaxf(mm, __shfl_xor(mm, off, kWave));
  if (WAVES > 1) {
    if ((tid & 63) == 0) sM[tid >> 6] = mm;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) mm = fmaxf(mm, sM[w]);
  }
  const float base = mm == -INFINITY ? 0.f : mm;
  float L = 0.f;
  for (int i = tid; i < n; i += WAVES * 64) {
    const float2 ml = part.ml[slot(i)];
    const float f = exp2f(ml.x - base);
    sF[i] = f;
    L += f * ml.y;
  }
  L = warp_sum(L);
  if ((tid & 63) == 0) sL[tid >> 6] = L;
  __syncthreads();
  L = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) L += sL[w];
  if (g < G) {
    floatx4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (g + u * G < n) O += sF[g + u * G] * x[u];
    for (int i = g + AHEAD * G; i < n; i += G) O += sF[i] * reinterpret_cast<const floatx4*>(part.o + slot(i) * D)[l4];
    sO[g][l4] = O;
  }
  __syncthreads();
  // (f16 parts' weights are 2^kLift times theirs, their sums too)
  if (tid == 0 && lse) lse[pair] = L == 0.f ? -INFINITY : (mm + log2f(L) - kLift<T>) * 0.69314718055994531f;
  if (tid >= L4) return;
  floatx4 O = sO[0][tid];
#pragma unroll
  for (int w = 1; w < G; ++w) O += sO[w][tid];
  const float inv = 1.f / L;
  T* out = reinterpret_cast<T*>(a.out) + row * a.o_row + h * a.o_head + 4 * tid;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(L == 0.f ? 0.f : O[e] * inv);
}

template <typename T, int D>
void launch_prefix(PrefixArgs a, const PrefixPlan& plan, void* workspace, float* lse, hipStream_t s) {
  a.own = plan.own;
  a.step = shared_step(D, sizeof(T) == 4);
  a.shared_blocks = plan.shared_blocks;
  a.blocks = plan.blocks;
  a.pairs = (size_t)a.r.rows * a.q_heads;
  const size_t n = a.pairs * plan.slots();
  Parts part;
  part.o = static_cast<float*>(workspace);
  part.ml = reinterpret_cast<float2*>(part.o + n * D);
  part.n = reinterpret_cast<int32_t*>(part.ml + n);
  launch_tiles<T, D>(a, plan.shared, part, attend_grid(plan.blocks), s);
  const dim3 grid(a.r.rows, a.q_heads);
  if (plan.slots() <= kJoinFew)
    hipLaunchKernelGGL((join_kernel<T, D, 1>), grid, dim3(64), 0, s, a, plan.shared.splits, part, lse);
  else
    hipLaunchKernelGGL((join_kernel<T, D, 4>), grid, dim3(256), 0, s, a, plan.shared.splits, part, lse);
  attend_launched(hipGetLastError());
}

template <typename T>
void launch_prefix_dim(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s) {
  switch (D) {
    case 32: return launch_prefix<T, 32>(a, plan, workspace, lse, s);
    case 64: return launch_prefix<T, 64>(a, plan, workspace, lse, s);
    case 96: return launch_prefix<T, 96>(a, plan, workspace, lse, s);
    case 128: return launch_prefix<T, 128>(a, plan, workspace, lse, s);
    case 192: return launch_prefix<T, 192>(a, plan, workspace, lse, s);
    case 256: return launch_prefix<T, 256>(a, plan, workspace, lse, s);
  }
}

#endif  // KV_ATTEND_KERNELS

}  // namespace mit2hip
