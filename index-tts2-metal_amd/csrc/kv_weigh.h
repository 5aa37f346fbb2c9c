// kv_weigh.h -- the attention weight that cached rows get (mit2cfm_kv_weigh): the
// kernel of one element type, instantiated in kv_weigh_{f32,f16,bf16}.hip.
#pragma once

#include "kv_attend.h"

namespace mit2hip {

struct WeighArgs {
  AttendArgs a;  // cache, rows, queries, mask (no output)
  float c2;      // scale log2(e)
  const float* lse;
  const float* weights;
  float* weights_out;
  int64_t stride;  // of a key head's weights
  float decay;
  int last_rows;  // 0: all
  const int32_t* position;
  int32_t* born;
};

void launch_weigh_f32(const WeighArgs& w, const WeighPlan& plan, int D, hipStream_t s);
void launch_weigh_f16(const WeighArgs& w, const WeighPlan& plan, int D, hipStream_t s);
void launch_weigh_bf16(const WeighArgs& w, const WeighPlan& plan, int D, hipStream_t s);

#if defined(KV_ATTEND_KERNELS)

// A query's operands, as load_query's.
template <typename T, int D>
__device__ __forceinline__ void load_row(const T* q, bool wide, int grp, typename Mat<T>::op (&qv)[Dims<T, D>::DC]) {
  typedef typename Mat<T>::op Op;
  constexpr int DC = Dims<T, D>::DC;
  if (wide) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int c = 0; c < DC; ++c) qv[c] = *reinterpret_cast<const Op*>(q + 32 * c + 8 * grp);
    } else {
#pragma unroll
      for (int c = 0; c < DC; c += 4) {
        const float4 x = *reinterpret_cast<const float4*>(q + D / 4 * grp + c);
        qv[c] = x.x; qv[c + 1] = x.y; qv[c + 2] = x.z; qv[c + 3] = x.w;
      }
    }
  } else {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int c = 0; c < DC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) qv[c][e] = q[32 * c + 8 * grp + e];
    } else {
#pragma unroll
      for (int c = 0; c < DC; ++c) qv[c] = q[D / 4 * grp + c];
    }
  }
}

// A wave holds 16 NT keys as operands and goes over query tiles of 16 (a sequence's
// new rows x the query heads of a key head): S = Q K^T leaves a lane four queries,
// from 4 (lane / 16) on, of key lane % 16 of each 16, and it adds up their weights
// exp2(scale2 s - log2(e) lse) in fp32; the four lanes of a key join at the end of the
// queries, two exchanges for each 16 keys.  BYQ: the block's four waves have the
// same keys and every fourth query tile each, and join in LDS, in order; else
// each wave goes over keys of its own.  No place is added to by two waves.
//
// Waves of their own keys: the cache's bytes bound it, 64 tokens over up to 8191 bf16 keys of
// 128 in 8 heads 164 us, 4.75 TB/s.  Shared keys: the products and exponentials, 16 prompts of
// 1029 rows, 32 heads, over 2047 f16 keys 319 us, 650 TFLOP/s.
//
// The third block of a CU is worth the few registers that 16-bit rows of 256 bytes spill
// for it: 4 ragged prompts of 1029 rows 70 us for 80, even ones 107 for 110 (of 512 rows 67
// for 63), 16 even ones 319 for 369; f32 rows, bound by their products, lose.
template <typename T, int D, bool BYQ>
__global__ __launch_bounds__(kAttendThreads, (BYQ && sizeof(T) == 2 && D <= 128) ? 3 : 2) void weigh_kernel(WeighArgs w, WeighPlan plan) {
  typedef Dims<T, D> S;
  typedef typename Mat<T>::op Op;
  constexpr int DC = S::DC, NT = weigh_tiles(D, sizeof(T)), KEYS = 16 * NT;
  __shared__ float sW[kAttendWaves][KEYS];
  constexpr bool STAGED = BYQ && D * sizeof(T) <= 256 && (D & (D - 1)) == 0;
  constexpr int CPR = D * sizeof(T) / 16, XM = CPR < 16 ? CPR - 1 : 15, LOADS = CPR / 4;  // a row's 16 bytes; a tile's loads
  constexpr int PLACES = STAGED ? 16 * CPR : 1;
  __shared__ __attribute__((aligned(1024))) u32x4 sQ0[kAttendWaves][PLACES], sQ1[kAttendWaves][PLACES], sQ2[kAttendWaves][PLACES];
  __shared__ __attribute__((aligned(16))) float sL0[kAttendWaves][16], sL1[kAttendWaves][16], sL2[kAttendWaves][16];
  const AttendArgs& a = w.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 15, grp = lane >> 4;
  Part p;
  uint32_t block = blockIdx.x;
  p.seq = blockIdx.z;
  p.kvh = blockIdx.y;
  if (plan.by_xcd) {  // workgroups go to the 8 XCDs in turn
    const uint32_t slot = block >> 3, line = slot / plan.blocks * 8 + (block & 7);
    block = slot % plan.blocks;
    p.seq = line / a.c.kv_heads;
    p.kvh = line - p.seq * a.c.kv_heads;
    if (p.seq >= a.r.seqs) return;
  }
  p.raw_start = a.r.start[p.seq];
  const int stop = a.r.start[p.seq + 1], length = a.r.length[p.seq];
  p.start = max(p.raw_start, 0);
  p.mrows = (min(stop, a.r.rows) - p.start) * a.group;
  if (p.mrows <= 0) return;
  p.first = length - (stop - p.raw_start);
  p.len = (int)min((int64_t)min(length, a.c.capacity()), w.stride);
  // query rows before this one are not counted
  const int from = w.last_rows ? (int)min(max((int64_t)stop - w.last_rows - p.start, (int64_t)0) * a.group, (int64_t)p.mrows) : 0;
  const int i0 = p.start - p.raw_start;  // place of query row 0 among the new rows
  const int32_t* table = a.c.table + (size_t)p.seq * a.c.table_stride;
  const T* K = reinterpret_cast<const T*>(a.c.k) + p.kvh * a.c.head_stride(D);
  const int64_t line = ((int64_t)p.seq * a.c.kv_heads + p.kvh) * w.stride;
  const T* const q0 = reinterpret_cast<const T*>(a.q) + p.start * a.q_row + p.kvh * a.group * a.q_head;
  const float* const lse0 = w.lse + (int64_t)p.start * a.q_heads + p.kvh * a.group;
  // From a lane's query to its next tile's: so many rows and heads on, or, past the
  // last head, one row more and the heads back.
  constexpr int STEP = BYQ ? 16 * kAttendWaves : 16;
  const int step_rows = STEP / a.group, step_heads = STEP - step_rows * a.group;
  const int64_t step_q = step_rows * a.q_row + step_heads * a.q_head, wrap_q = a.q_row - a.group * a.q_head;
  const int step_lse = step_rows * a.q_heads + step_heads, wrap_lse = a.q_heads - a.group;

  const int64_t each = BYQ ? KEYS : KEYS * kAttendWaves;
  int entry[NT];  // of this lane's keys' pages
  auto look_up = [&](int64_t j0) {
#pragma unroll
    for (int t = 0; t < NT; ++t) entry[t] = table[min(j0 + 16 * t + lq, (int64_t)p.len - 1) >> a.c.page_shift];
  };
  int64_t b0 = block * each;
  if (b0 >= p.len) return;
  look_up(b0 + (BYQ ? 0 : KEYS * wave));
  for (; b0 < p.len; b0 += plan.blocks * each) {
    const int64_t j0_ = b0 + (BYQ ? 0 : KEYS * wave);
    if (!BYQ && j0_ >= p.len) break;
    const int j0 = (int)j0_;
    bool there[NT], all_there = true;
    Op kv[NT][DC];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int j = j0 + 16 * t + lq;
      there[t] = j < p.len && (unsigned)entry[t] < (unsigned)a.c.pages;
      all_there = all_there && there[t];
      const T* kp = K + a.c.row_in(there[t] ? entry[t] : 0, j, D);
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
    // this lane's place, and what it had before
    const int place = BYQ ? j0 + tid : j0 + lane;
    const bool writes = (BYQ ? tid : lane) < KEYS && place < p.len;
    float old = 0.f;
    if (writes && place < p.first) old = w.weights[line + place];
    if (!BYQ && b0 + plan.blocks * each + KEYS * wave < p.len) look_up(b0 + plan.blocks * each + KEYS * wave);
    all_there = !__any(!all_there);

    // a chain's rows before the wave's first key see none of them
    int m0 = from;
    if (!a.mask) m0 = (int)min(max((int64_t)from, ((int64_t)j0 - p.first - i0) * a.group), (int64_t)p.mrows);
    m0 = from + (m0 - from) / 16 * 16;
    if (BYQ) m0 += 16 * wave;
    int first_row = m0 / a.group, first_head = m0 - first_row * a.group;  // of the tile's first query
    int row = (m0 + lq) / a.group, g = m0 + lq - row * a.group;           // this lane's of 16
    int64_t at_q = row * a.q_row + g * a.q_head;
    int at_lse = row * a.q_heads + g;

    float acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = 0.f;
    // A tile's queries: operands, log sum and row of this lane's (past the last one: the
    // first, as one that sees nothing).
    struct Tile {
      Op q[DC];
      float lse;
      int row;
    };
    auto fetch = [&](int m, Tile& x) {
      const bool whole = m + 16 <= p.mrows, ok = m + lq < p.mrows;
      load_row<T, D>(q0 + (whole || ok ? at_q : 0), a.q_wide, grp, x.q);
      x.lse = lse0[whole || ok ? at_lse : 0];
      x.row = row;
      if (!whole) {
        x.lse = ok ? x.lse : -INFINITY;
        x.row = ok ? row : 0;
      }
      row += step_rows;
      at_q += step_q;
      at_lse += step_lse;
      if (step_heads) {
        g += step_heads;
        const bool wrap = g >= a.group;
        g -= wrap ? a.group : 0;
        row += wrap ? 1 : 0;
        at_q += wrap ? wrap_q : 0;
        at_lse += wrap ? wrap_lse : 0;
      }
    };
    // A tile's weights: its operands, log2 sums and rows (y(r)) of the lane's four queries.
    auto weigh = [&](const Op(&q)[DC], const float(&base)[4], bool sightless, auto&& y_of) {
      // all the tile's rows see all the wave's keys?
      const bool open = j0 + KEYS <= p.first || (!a.mask && j0 + KEYS - 1 - p.first <= i0 + first_row);
      const bool some = !open || !all_there || sightless;
      first_head += step_heads;
      first_row += step_rows + (first_head >= a.group ? 1 : 0);
      first_head -= first_head >= a.group ? a.group : 0;
      floatx4 x[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) x[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DC; ++d)
#pragma unroll
        for (int t = 0; t < NT; ++t) x[t] = Mat<T>::mul(q[d], kv[t][d], x[t]);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[t][r] = __builtin_amdgcn_exp2f(fmaf(x[t][r], w.c2, base[r]));
      if (some) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int y = y_of(r);
          const bool lives = base[r] != -INFINITY;
          const uint32_t* words = a.mask + (int64_t)(p.start + y) * a.mask_words;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const int n = j0 + 16 * t + lq - p.first;  // the key's place among the new rows
            uint32_t sees = n <= i0 + y ? 1u : 0u;
            if (a.mask) {
              const int word = n >> 5;
              sees = words[min(max(word, 0), a.mask_words - 1)] >> (n & 31) & 1u;
              sees = n < 0 ? 1u : word < a.mask_words ? sees : 0u;
            }
            x[t][r] = sees && lives && there[t] ? x[t][r] : 0.f;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] += (x[t][0] + x[t][1]) + (x[t][2] + x[t][3]);
    };
    if constexpr (STAGED) {
      if (a.q_wide) {
        // Through LDS, a ring of the wave's own: 16 lanes read a row's neighbouring 16 bytes
        // each.  (Straight into operands each lane is in a row of its own, and the loads'
        // 64 addresses a third of the time: 16 prompts of 1029 rows over 2047 f16 keys 480 us
        // so, 374 through LDS, both at two blocks a CU.)  Three tiles, objects of their own so that a read waits
        // for its own alone, two ahead; tiles past the end are the last one again, so that
        // the loads in flight are always as many.
        const int o0 = lane / CPR, place16 = lane % CPR;
        constexpr int ROWS = 64 / CPR;  // a load's rows
        const T* at[LOADS];             // this lane's of the next tile
        int at_g[LOADS], lse_g = 0;
        const float* at_l = lse0;
        auto point = [&](int m, int u) {  // (rows past the last one: the last one)
          const int o = o0 + ROWS * u, x = min(m + o, p.mrows - 1), n = x / a.group;
          at_g[u] = x - n * a.group;
          at[u] = q0 + n * a.q_row + at_g[u] * a.q_head + (place16 ^ (o & XM)) * (16 / (int)sizeof(T));
        };
        auto point_lse = [&](int m) {
          const int x = min(m + lq, p.mrows - 1), n = x / a.group;
          lse_g = x - n * a.group;
          at_l = lse0 + n * a.q_heads + lse_g;
        };
        auto stage = [&](int m, u32x4* to, float* to_lse) {
          if (m + 16 > p.mrows) {
#pragma unroll
            for (int u = 0; u < LOADS; ++u) point(m, u);
            point_lse(m);
          }
#pragma unroll
          for (int u = 0; u < LOADS; ++u) load_to_lds(at[u], (lds_ptr_t*)(to + 64 * u));
          if (lane < 16) load4_to_lds(at_l, (lds_ptr_t*)to_lse);
#pragma unroll
          for (int u = 0; u < LOADS; ++u) at[u] += step_q;
          at_l += step_lse;
          if (step_heads) {
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
              at_g[u] += step_heads;
              at[u] += at_g[u] >= a.group ? wrap_q : 0;
              at_g[u] -= at_g[u] >= a.group ? a.group : 0;
            }
            lse_g += step_heads;
            at_l += lse_g >= a.group ? wrap_lse : 0;
            lse_g -= lse_g >= a.group ? a.group : 0;
          }
        };
        auto use = [&](int m, const u32x4* tile, const float* tile_lse) {
          wait_loads<2 * (LOADS + 1)>();
          __asm__ volatile("" ::: "memory");
          Op q[DC];
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int c = 0; c < DC; ++c) q[c] = *reinterpret_cast<const Op*>(&tile[lq * CPR + ((4 * c + grp) ^ (lq & XM))]);
          } else {
#pragma unroll
            for (int c = 0; c < DC; c += 4) {
              const floatx4 x = *reinterpret_cast<const floatx4*>(&tile[lq * CPR + ((DC / 4 * grp + c / 4) ^ (lq & XM))]);
              q[c] = x[0]; q[c + 1] = x[1]; q[c + 2] = x[2]; q[c + 3] = x[3];
            }
          }
          const floatx4 l = *reinterpret_cast<const floatx4*>(tile_lse + 4 * grp);
          float base[4];
          bool sightless = m + 16 > p.mrows;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool dead = l[r] == -INFINITY || m + 4 * grp + r >= p.mrows;
            base[r] = dead ? -INFINITY : l[r] * -1.4426950408889634f;
            sightless = sightless || dead;
          }
          weigh(q, base, __any(sightless), [&](int r) { return min(m + 4 * grp + r, p.mrows - 1) / a.group; });
        };
        if (m0 < p.mrows) {
          u32x4 *q0s = sQ0[wave], *q1s = sQ1[wave], *q2s = sQ2[wave];
#pragma unroll
          for (int u = 0; u < LOADS; ++u) point(m0, u);
          point_lse(m0);
          stage(m0, q0s, sL0[wave]);
          stage(m0 + STEP, q1s, sL1[wave]);
          wait_loads<2 * (LOADS + 1)>();  // (the keys are here: no wait for them in the loop)
          for (int m = m0;;) {
            stage(m + 2 * STEP, q2s, sL2[wave]);
            use(m, q0s, sL0[wave]);
            if ((m += STEP) >= p.mrows) break;
            stage(m + 2 * STEP, q0s, sL0[wave]);
            use(m, q1s, sL1[wave]);
            if ((m += STEP) >= p.mrows) break;
            stage(m + 2 * STEP, q1s, sL1[wave]);
            use(m, q2s, sL2[wave]);
            if ((m += STEP) >= p.mrows) break;
          }
          wait_loads<0>();  // (the ring is filled again for the next keys)
        }
        m0 = p.mrows;
      }
    }
    auto one_by_one = [&](const Tile& q) {
      // (a row that sees nothing: -inf)
      const float mine = q.lse == -INFINITY ? -INFINITY : q.lse * -1.4426950408889634f;
      float base[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) base[r] = __shfl(mine, 4 * grp + r, kWave);
      weigh(q.q, base, __any(mine == -INFINITY), [&](int r) { return __shfl(q.row, 4 * grp + r, kWave); });
    };
    Tile one;
    if constexpr (STAGED) {
      for (int m = m0; m < p.mrows; m += STEP) {
        fetch(m, one);
        one_by_one(one);
      }
    } else {
      // (two tiles in turn, each asked for during the other)
      Tile other;
      if (m0 < p.mrows) fetch(m0, one);
      for (int m = m0; m < p.mrows; m += 2 * STEP) {
        if (m + STEP < p.mrows) fetch(m + STEP, other);
        one_by_one(one);
        if (m + STEP >= p.mrows) break;
        if (m + 2 * STEP < p.mrows) fetch(m + 2 * STEP, one);
        one_by_one(other);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      acc[t] += __shfl_xor(acc[t], 16, kWave);
      acc[t] += __shfl_xor(acc[t], 32, kWave);
    }
    float sum = acc[0];  // of key `lane`
    if (BYQ) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (grp == t % 4) sW[wave][16 * t + lq] = acc[t];
      __syncthreads();
      if (writes) {
        sum = sW[0][tid];
#pragma unroll
        for (int v = 1; v < kAttendWaves; ++v) sum += sW[v][tid];
      }
    } else {
#pragma unroll
      for (int t = 1; t < NT; ++t) sum = grp == t ? acc[t] : sum;
    }
    if (writes) {
      // (a product and a sum, each rounded)
      w.weights_out[line + place] = place < p.first ? __fadd_rn(__fmul_rn(w.decay, old), sum) : sum;
      if (w.born && place >= p.first) {
        const int64_t row = (int64_t)p.raw_start + (place - p.first);
        if (!w.position)
          w.born[line + place] = place;
        else if (row >= 0 && row < a.r.rows)
          w.born[line + place] = w.position[row];
      }
    }
    if (BYQ) {
      __syncthreads();
      if (b0 + plan.blocks * each < p.len) look_up(b0 + plan.blocks * each);
    }
  }
}

template <typename T, int D>
void launch_weigh(const WeighArgs& w, const WeighPlan& plan, hipStream_t s) {
  const uint32_t lines = (uint32_t)w.a.c.kv_heads * w.a.r.seqs;
  const uint32_t x = weigh_grid(plan, lines);
  const dim3 grid = plan.by_xcd ? dim3(x) : dim3(x, w.a.c.kv_heads, w.a.r.seqs);
  const dim3 block(kAttendThreads);
  if (plan.by_query)
    hipLaunchKernelGGL((weigh_kernel<T, D, true>), grid, block, 0, s, w, plan);
  else
    hipLaunchKernelGGL((weigh_kernel<T, D, false>), grid, block, 0, s, w, plan);
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
