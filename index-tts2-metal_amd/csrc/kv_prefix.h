// kv_prefix.h -- attention of sequences that share their first rows
// (mit2cfm_kv_prefix_attention): the launches of one element type, instantiated in
// kv_prefix_{f32,f16,bf16}.hip.
#pragma once

#include "kv_attend.h"

namespace mit2hip {

// How the two halves are laid out.
struct PrefixPlan {
  AttendPlan shared, own;
  bool shares;  // there may be shared rows
  int slots() const { return (shares ? shared.splits : 0) + own.splits; }
};
inline PrefixPlan prefix_plan(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads, const mit2cfm_kv_prefix& x) {
  PrefixPlan p{};
  p.shares = x.groups > 0;
  mit2cfm_kv_rows some = r;
  if (p.shares) {
    some.seqs = x.groups;
    some.max_length = x.max_shared;
    p.shared = attend_plan(c, some, q_heads);
  }
  some.seqs = r.seqs;
  some.max_length = !p.shares ? r.max_length : r.max_length > x.max_shared ? r.max_length - x.max_shared + 63 : 64;
  p.own = attend_plan(c, some, q_heads);
  return p;
}

// Launches both halves and their join; throws HipError.  lse may be NULL.
void launch_prefix_f32(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s);
void launch_prefix_f16(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s);
void launch_prefix_bf16(const PrefixArgs& a, const PrefixPlan& plan, int D, void* workspace, float* lse, hipStream_t s);

#if defined(KV_ATTEND_KERNELS)

// Joins the parts of a row and query head, a wave each: those of the shared rows, then
// its sequence's own.  Lane groups of D/4 take every so manyth part, four elements a lane.
template <typename T, int D>
__global__ __launch_bounds__(64) void join_kernel(PrefixArgs a, Parts part, const int32_t* shared_parts, float* lse) {
  constexpr int L4 = D / 4, G = 64 / L4;
  __shared__ floatx4 sO[G][L4];
  __shared__ float sF[2 * kMostSplits];
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  if (row < a.r.start[0] || row >= a.r.start[a.r.seqs]) return;  // nobody's row
  const size_t pair = (size_t)row * a.q_heads + h, at = pair * a.slots;
  const int told = part.n[pair], shared = told >> 16 ? min(max(shared_parts[pair], 0), a.slot0) : 0;
  const int n = shared + min(told & 0xffff, a.slots - a.slot0);
  auto slot = [&](int i) { return at + (i < shared ? i : a.slot0 + i - shared); };
  float mm = -INFINITY;
  for (int i = tid; i < n; i += 64) mm = fmaxf(mm, part.ml[slot(i)].x);
#pragma unroll
  for (int off = 32; off; off >>= 1) mm = fmaxf(mm, __shfl_xor(mm, off, kWave));
  const float base = mm == -INFINITY ? 0.f : mm;
  float L = 0.f;
  for (int i = tid; i < n; i += 64) {
    const float2 ml = part.ml[slot(i)];
    const float f = exp2f(ml.x - base);
    sF[i] = f;
    L += f * ml.y;
  }
  L = warp_sum(L);
  __syncthreads();
  const int g = tid / L4, l4 = tid - g * L4;
  if (g < G) {
    floatx4 O = {0.f, 0.f, 0.f, 0.f};
    for (int i = g; i < n; i += G) O += sF[i] * reinterpret_cast<const floatx4*>(part.o + slot(i) * D)[l4];
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
  a.slots = plan.slots();
  const size_t pairs = (size_t)a.r.rows * a.q_heads, n = pairs * a.slots;
  Parts part;
  part.o = static_cast<float*>(workspace);
  part.ml = reinterpret_cast<float2*>(part.o + n * D);
  part.n = reinterpret_cast<int32_t*>(part.ml + n);
  int32_t* const own_parts = part.n + pairs;
  if (plan.shares) {
    a.own = 0;
    a.slot0 = 0;
    launch_tiles<T, D>(a, plan.shared, part, s);
  }
  const int32_t* shared_parts = part.n;
  part.n = own_parts;
  a.own = 1;
  a.slot0 = a.slots - plan.own.splits;
  launch_tiles<T, D>(a, plan.own, part, s);
  hipLaunchKernelGGL((join_kernel<T, D>), dim3(a.r.rows, a.q_heads), dim3(64), 0, s, a, part, shared_parts, lse);
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
