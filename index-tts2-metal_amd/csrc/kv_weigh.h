// kv_weigh.h -- the attention weight that cached rows get (mit2cfm_kv_weigh): the
// kernel of one element type, instantiated in kv_weigh_{f32,f16,bf16}.hip.
#pragma once

#include "kv_attend.h"

namespace mit2hip {

struct WeighArgs {
  AttendArgs a;  // cache, rows, queries, mask, scale (no output)
  const float* lse;
  const float* weights;
  float* weights_out;
  int64_t stride;  // of a key head's weights
  float decay;
  int last_rows;  // 0: all
  const int32_t* position;
  int32_t* born;
};

// Whether a block's waves share their keys and divide the queries (kv_weigh.hip).
struct WeighPlan {
  int by_query;
  uint32_t chunks;  // blocks of a sequence and key head
};

void launch_weigh_f32(const WeighArgs& w, const WeighPlan& plan, int D, hipStream_t s);
void launch_weigh_f16(const WeighArgs& w, const WeighPlan& plan, int D, hipStream_t s);
void launch_weigh_bf16(const WeighArgs& w, const WeighPlan& plan, int D, hipStream_t s);

// 16-key tiles of a wave: up to 64 keys, 16 KB of them.
constexpr int weigh_tiles(int D, int bytes) { return D * bytes <= 256 ? 4 : D * bytes <= 512 ? 2 : 1; }

#if defined(KV_ATTEND_KERNELS)

// A wave holds 16 NT keys as operands and goes over query tiles of 16 (a sequence's
// new rows x the query heads of a key head): S^T = K Q^T leaves a lane one query
// and four keys of each 16, whose weights exp2(scale2 s - log2(e) lse) it adds up in
// fp32, tile after tile; its 16 queries' sums are joined at the end.  BYQ: the block's four
// waves have the same keys and every fourth query tile each, and join in LDS, in
// order; else each wave has keys of its own.  No place is added to by two blocks.
template <typename T, int D, bool BYQ>
__global__ __launch_bounds__(kAttendThreads) void weigh_kernel(WeighArgs w, uint32_t chunks) {
  typedef Dims<T, D> S;
  typedef typename Mat<T>::op Op;
  constexpr int DC = S::DC, NT = weigh_tiles(D, sizeof(T)), KEYS = 16 * NT, NV = 4 * NT;
  constexpr int BLOCK_KEYS = BYQ ? KEYS : KEYS * kAttendWaves;
  __shared__ float sW[kAttendWaves][KEYS];
  const AttendArgs& a = w.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 15, grp = lane >> 4;
  Part p;
  p.seq = blockIdx.z;
  p.kvh = blockIdx.y;
  p.raw_start = a.r.start[p.seq];
  const int stop = a.r.start[p.seq + 1], length = a.r.length[p.seq];
  p.start = max(p.raw_start, 0);
  p.mrows = (min(stop, a.r.rows) - p.start) * a.group;
  if (p.mrows <= 0) return;
  p.first = length - (stop - p.raw_start);
  p.len = (int)min((int64_t)min(length, a.c.capacity()), w.stride);
  // query rows before this one are not counted
  const int from = w.last_rows ? (int)min(max((int64_t)stop - w.last_rows - p.start, (int64_t)0) * a.group, (int64_t)p.mrows) : 0;
  const int32_t* table = a.c.table + (size_t)p.seq * a.c.table_stride;
  const T* K = reinterpret_cast<const T*>(a.c.k) + p.kvh * a.c.head_stride(D);
  const int64_t line = ((int64_t)p.seq * a.c.kv_heads + p.kvh) * w.stride;

  for (int64_t c = blockIdx.x; c * BLOCK_KEYS < p.len; c += chunks) {
    const int b0 = (int)c * BLOCK_KEYS, j0 = BYQ ? b0 : b0 + KEYS * wave;
    float acc[NV];
#pragma unroll
    for (int e = 0; e < NV; ++e) acc[e] = 0.f;
    if (j0 < p.len) {
      int page[NT];
      uint32_t there = 0;  // bit e: this lane's key e is
#pragma unroll
      for (int t = 0; t < NT; ++t) page[t] = table[min(j0 + 16 * t + lq, p.len - 1) >> a.c.page_shift];
      Op kv[NT][DC];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int j = j0 + 16 * t + lq;
        const bool ok = j < p.len && (unsigned)page[t] < (unsigned)a.c.pages;
        there |= ((uint32_t)(__ballot(ok) >> (4 * grp)) & 15u) << (4 * t);
        const T* kp = K + a.c.row_in(ok ? page[t] : 0, j, D);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int d = 0; d < DC; ++d) kv[t][d] = *reinterpret_cast<const Op*>(kp + 32 * d + 8 * grp);
        } else {
#pragma unroll
          for (int d = 0; d < DC; d += 4) {
            const float4 x = *reinterpret_cast<const float4*>(kp + D / 4 * grp + d);
            kv[t][d] = x.x; kv[t][d + 1] = x.y; kv[t][d + 2] = x.z; kv[t][d + 3] = x.w;
          }
        }
      }
      const bool all_there = !__any(there != (1u << NV) - 1u);
      // a chain's rows before the wave's first key see none of them
      const int i0 = p.start - p.raw_start;  // place of query row 0 among the new rows
      int m0 = from;
      if (!a.mask) m0 = (int)min(max((int64_t)from, ((int64_t)j0 - p.first - i0) * a.group), (int64_t)p.mrows);
      m0 = from + (m0 - from) / 16 * 16;
      constexpr int STEP = BYQ ? 16 * kAttendWaves : 16;
      if (BYQ) m0 += 16 * wave;

      Op next[DC];
      float lse_next = 0.f;
      auto fetch = [&](int m) {
        const Query x(a, p, min(m + lq, p.mrows - 1));
        load_query<T, D>(a, x, grp, next);
        lse_next = w.lse[(int64_t)x.row * a.q_heads + x.h];
      };
      if (m0 < p.mrows) fetch(m0);
      for (int m = m0; m < p.mrows; m += STEP) {
        Op qv[DC];
#pragma unroll
        for (int d = 0; d < DC; ++d) qv[d] = next[d];
        const float lse = lse_next;
        const bool live = m + lq < p.mrows && lse != -INFINITY;
        if (m + STEP < p.mrows) fetch(m + STEP);
        uint32_t seen = there;
        // all the tile's rows see all the wave's keys?
        const int least = (p.start + m / a.group) - p.raw_start;  // the tile's first row among the new ones
        const bool open = j0 + KEYS <= p.first || (!a.mask && j0 + KEYS - 1 - p.first <= least);
        if (!open) seen = seen_keys<NV>(a, Query(a, p, min(m + lq, p.mrows - 1)), j0, p.first, grp, there);
        if (!live) seen = 0;
        const bool some = !open || !all_there || __any(!live);
        const float base = -lse * 1.4426950408889634f;
        float s[NV];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int d = 0; d < DC; ++d) x = Mat<T>::mul(kv[t][d], qv[d], x);
#pragma unroll
          for (int r = 0; r < 4; ++r) s[4 * t + r] = x[r];
        }
#pragma unroll
        for (int e = 0; e < NV; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale2, base));
        if (some) {
#pragma unroll
          for (int e = 0; e < NV; ++e) s[e] = seen >> e & 1u ? s[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < NV; ++e) acc[e] += s[e];
      }
    }
#pragma unroll
    for (int e = 0; e < NV; ++e) {
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) acc[e] += __shfl_xor(acc[e], off, kWave);
    }
    if (lq == 0) {
#pragma unroll
      for (int e = 0; e < NV; ++e) sW[wave][key_of(e, grp)] = acc[e];
    }
    __syncthreads();
    if (tid < BLOCK_KEYS && b0 + tid < p.len) {
      const int j = b0 + tid;
      float sum;
      if (BYQ) {
        sum = sW[0][tid % KEYS];
#pragma unroll
        for (int v = 1; v < kAttendWaves; ++v) sum += sW[v][tid % KEYS];
      } else {
        sum = sW[tid / KEYS][tid % KEYS];
      }
      // (a product and a sum, each rounded)
      w.weights_out[line + j] = j < p.first ? __fadd_rn(__fmul_rn(w.decay, w.weights[line + j]), sum) : sum;
      if (w.born && j >= p.first) {
        const int64_t row = (int64_t)p.raw_start + (j - p.first);
        if (!w.position)
          w.born[line + j] = j;
        else if (row >= 0 && row < a.r.rows)
          w.born[line + j] = w.position[row];
      }
    }
    __syncthreads();
  }
}

template <typename T, int D>
void launch_weigh(const WeighArgs& w, const WeighPlan& plan, hipStream_t s) {
  const dim3 grid(plan.chunks, w.a.c.kv_heads, w.a.r.seqs), block(kAttendThreads);
  if (plan.by_query)
    hipLaunchKernelGGL((weigh_kernel<T, D, true>), grid, block, 0, s, w, plan.chunks);
  else
    hipLaunchKernelGGL((weigh_kernel<T, D, false>), grid, block, 0, s, w, plan.chunks);
  attend_launched(hipGetLastError());
}

template <typename T>
void launch_weigh_dim(const WeighArgs& w, const WeighPlan& plan, int D, hipStream_t s) {
  switch (D) {
    case 32: return launch_weigh<T, 32>(w, plan, s);
    case 64: return launch_weigh<T, 64>(w, plan, s);
    case 96: return launch_weigh<T, 96>(w, plan, s);
    case 128: return launch_weigh<T, 128>(w, plan, s);
    case 192: return launch_weigh<T, 192>(w, plan, s);
    case 256: return launch_weigh<T, 256>(w, plan, s);
  }
}

#endif  // KV_ATTEND_KERNELS

}  // namespace mit2hip
