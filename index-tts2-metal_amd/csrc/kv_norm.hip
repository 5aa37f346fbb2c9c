// kv_norm.hip -- the append whose query and key heads are normalised before they
// are rotated (see kv_ops.h and mit2cfm.h for what it computes).
#include <cfloat>
#include <cmath>

#include "kv_args.h"

namespace mit2hip {

namespace {

constexpr int kNormThreads = 256;

struct NormArgs {
  AppendArgs a;
  const char *q_weight, *k_weight;
  int64_t qw_head, kw_head;
  int f32_weight, centered;
  float eps;
};

// The sum over G neighbouring lanes (a power of two, in a wave), in all of them.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = 1; off < G; off <<= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// A group of G lanes takes a head, its items (as the plain append's: two vectors of
// VEC elements that hold both elements of each rotated pair) a lane's each, NI
// at most; blockIdx.y: a block's share of a row's heads.  The elements stay in
// registers, in fp32, between the read and the one write: sums, mean, norm, weight
// and rotation are fp32, and rounded to the type at the end.
//
// The first heads are asked for before the row's sequence is known, and the angles'
// frequencies formed meanwhile (fp64, as the positions times them).
//
// 9 prompts of up to 2047 rows, 32 + 8 + 8 bf16 heads of 128: 67 us, 4.9 TB/s, as fast as
// a copy (5.0).  3 rows of 20 fp32 heads of 64: 4.4 us, the launch and the way to the row's page.
template <typename T, int VEC, int G, int NI>
__global__ __launch_bounds__(kNormThreads) void norm_append_kernel(NormArgs n, int D) {
  constexpr int HEADS = kNormThreads / G;  // heads of a pass
  __shared__ float2 turn[kMaxPairs];
  __shared__ int64_t s_at;  // element index of the row in its page, head 0; -1: not written
  __shared__ int s_place;   // the row's position
  __shared__ int s_mine;    // the row is a sequence's
  const AppendArgs& a = n.a;
  const int tid = threadIdx.x, row = blockIdx.x, lane = tid % G;
  const int half = a.rot >> 1, per_head = D / (2 * VEC);
  const int norm_heads = a.q_heads + a.c.kv_heads, heads = norm_heads + a.c.kv_heads;
  typedef Vec<T, VEC> V;

  // An item's two vectors, and the pair index of its first element.
  auto place = [&](int u, bool rotates, int& e0, int& e1, int& pair0) {
    if (a.interleaved || !rotates) {
      e0 = 2 * VEC * u;
      e1 = e0 + VEC;
      pair0 = VEC * u;
      return rotates && e0 < a.rot;
    }
    if (u * VEC < half) {
      e0 = pair0 = VEC * u;
      e1 = e0 + half;
      return true;
    }
    e0 = a.rot + 2 * (VEC * u - half);
    e1 = e0 + VEC;
    pair0 = 0;
    return false;
  };
  auto source = [&](int h) {
    if (h < a.q_heads) return reinterpret_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
    if (h < norm_heads) return reinterpret_cast<const T*>(a.k) + row * a.k_row + (h - a.q_heads) * a.k_head;
    return reinterpret_cast<const T*>(a.v) + row * a.v_row + (h - norm_heads) * a.v_head;
  };
  V x[NI], y[NI];
  auto read = [&](int h) {
    const T* src = source(h);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      int e0, e1, pair0;
      const int u = lane + i * G;
      if (u >= per_head) continue;
      place(u, h < norm_heads, e0, e1, pair0);
      x[i] = *reinterpret_cast<const V*>(src + e0);
      y[i] = *reinterpret_cast<const V*>(src + e1);
    }
  };

  const int step = gridDim.y * HEADS;
  int h = blockIdx.y * HEADS + tid / G;
  if (h < heads) read(h);
  double inv = 0.0;  // turns a position
  const int pair = tid - 64;
  if (tid < 64) {
    const int seq = seq_of_row(a.r, row);
    if (tid == 0) {
      int64_t at = -1;
      int pos = 0;
      if (seq >= 0) {
        const int place = a.r.length[seq] - (a.r.start[seq + 1] - row);
        if (place >= 0 && place < a.c.capacity()) {
          const int page = a.c.page_of(seq, place);
          if (page >= 0) at = a.c.row_in(page, place, D);
        }
        pos = a.position ? a.position[row] : place;
      }
      s_at = at;
      s_place = pos;
      s_mine = seq >= 0;
    }
  } else if (pair < half) {
    inv = exp2(-2.0 * pair / a.rot * a.log2_theta) * 0.15915494309189533577;  // 1 / (2 pi)
  }
  __syncthreads();
  if (!s_mine) return;
  if (pair >= 0 && pair < half) {
    double t = (double)s_place * inv;
    t -= rint(t);
    float sn, cs;
    sincospif((float)(2.0 * t), &sn, &cs);
    turn[pair] = make_float2(cs, sn);
  }
  __syncthreads();

  for (bool first = true; h < heads; h += step, first = false) {
    if (!first) read(h);
    T* dst;
    if (h < a.q_heads) {
      dst = reinterpret_cast<T*>(a.q_out) + row * a.qo_row + h * a.qo_head;
    } else {
      if (s_at < 0) continue;
      const bool is_k = h < norm_heads;
      dst = reinterpret_cast<T*>(is_k ? a.c.k : a.c.v) + s_at + (is_k ? h - a.q_heads : h - norm_heads) * a.c.head_stride(D);
    }
    if (h >= norm_heads) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int u = lane + i * G;
        if (u >= per_head) continue;
        *reinterpret_cast<V*>(dst + 2 * VEC * u) = x[i];
        *reinterpret_cast<V*>(dst + 2 * VEC * u + VEC) = y[i];
      }
      continue;
    }
    float fx[NI][VEC], fy[NI][VEC];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const bool in = lane + i * G < per_head;
        fx[i][j] = in ? (float)x[i].v[j] : 0.f;
        fy[i][j] = in ? (float)y[i].v[j] : 0.f;
      }
    // (x - mean) * by, and the mean of its squares; lanes without an item stay 0
    auto statistics = [&](float by) {
      if (n.centered) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) sum += fx[i][j] * by + fy[i][j] * by;
        return group_sum<G>(sum) / D;
      }
      return 0.f;
    };
    auto squares = [&](float by, float mean) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (lane + i * G < per_head) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float p = fx[i][j] * by - mean, q = fy[i][j] * by - mean;
            sum += p * p + q * q;
          }
        }
      return group_sum<G>(sum) / D;
    };
    float by = 1.f, mean = statistics(1.f), square = squares(1.f, mean);
    if (!(square <= FLT_MAX)) {  // squares past fp32's range (or NaN): of 2^-70 of the elements
      by = 0x1p-70f;
      mean = statistics(by);
      square = squares(by, mean);
    }
    const float scale = 1.f / sqrtf(square + n.eps * by * by);

    const bool is_q = h < a.q_heads;
    const char* weight = is_q ? n.q_weight : n.k_weight;
    const int64_t w0 = is_q ? h * n.qw_head : (h - a.q_heads) * n.kw_head;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int u = lane + i * G;
      if (u >= per_head) continue;
      int e0, e1, pair0;
      const bool turned = place(u, true, e0, e1, pair0);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        fx[i][j] = (fx[i][j] * by - mean) * scale;
        fy[i][j] = (fy[i][j] * by - mean) * scale;
      }
      if (weight) {
        if (n.f32_weight) {
          const float* w = reinterpret_cast<const float*>(weight) + w0;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            fx[i][j] *= w[e0 + j];
            fy[i][j] *= w[e1 + j];
          }
        } else {
          const T* w = reinterpret_cast<const T*>(weight) + w0;
          const V wx = *reinterpret_cast<const V*>(w + e0), wy = *reinterpret_cast<const V*>(w + e1);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            fx[i][j] *= (float)wx.v[j];
            fy[i][j] *= (float)wy.v[j];
          }
        }
      }
      if (turned) {
        if (a.interleaved) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            // pair j of the item: elements 2 j, 2 j + 1 of (x, y)
            float& p = 2 * j < VEC ? fx[i][(2 * j) % VEC] : fy[i][(2 * j) % VEC];
            float& q = 2 * j + 1 < VEC ? fx[i][(2 * j + 1) % VEC] : fy[i][(2 * j + 1) % VEC];
            if (pair0 + j < half) {
              const float2 cs = turn[pair0 + j];
              const float fp = p, fq = q;
              p = fp * cs.x - fq * cs.y;
              q = fq * cs.x + fp * cs.y;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float2 cs = turn[pair0 + j];
            const float fp = fx[i][j], fq = fy[i][j];
            fx[i][j] = fp * cs.x - fq * cs.y;
            fy[i][j] = fq * cs.x + fp * cs.y;
          }
        }
      }
      V rx, ry;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        rx.v[j] = (T)fx[i][j];
        ry.v[j] = (T)fy[i][j];
      }
      *reinterpret_cast<V*>(dst + e0) = rx;
      *reinterpret_cast<V*>(dst + e1) = ry;
    }
  }
}

template <typename T, int VEC, int G, int NI>
void launch_by(const NormArgs& n, int D, hipStream_t s) {
  constexpr int HEADS = kNormThreads / G;
  const int heads = n.a.q_heads + 2 * n.a.c.kv_heads;
  // few rows: their heads over more blocks, down to one a group of lanes (64 rows of 48
  // heads 4.6 us, with a block a row 5.9; 512 to 8192 blocks are alike)
  const int by = std::max(1, std::min((heads + HEADS - 1) / HEADS, 2048 / n.a.r.rows));
  hipLaunchKernelGGL((norm_append_kernel<T, VEC, G, NI>), dim3(n.a.r.rows, by), dim3(kNormThreads), 0, s, n, D);
  kv_launched(hipGetLastError());
}

template <typename T>
void launch(const NormArgs& n, int D, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](const void* p, int64_t head) { return aligned(p, 16) && head % V == 0; };
  if (!append_wide(n.a, V) || !fits(n.q_weight, n.qw_head) || !fits(n.k_weight, n.kw_head))
    return launch_by<T, 1, 64, 2>(n, D, s);
  const int items = D / (2 * V);  // lanes of a head: the next power of two
  if (items <= 2) return launch_by<T, V, 2, 1>(n, D, s);
  if (items <= 4) return launch_by<T, V, 4, 1>(n, D, s);
  if (items <= 8) return launch_by<T, V, 8, 1>(n, D, s);
  if (items <= 16) return launch_by<T, V, 16, 1>(n, D, s);
  launch_by<T, V, 32, 1>(n, D, s);
}

}  // namespace

void kv_norm_append(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, const mit2cfm_kv_append& p,
                    const mit2cfm_kv_norm& m, hipStream_t s) {
  NormArgs n;
  need(m.weight_dtype == MIT2CFM_DTYPE_F32 || m.weight_dtype == c.dtype, "weight_dtype must be f32 or the cache's");
  need(m.eps >= 1e-20f && m.eps <= 1e20f, "eps must be in [1e-20, 1e20]");
  if (!append_args(c, r, p, n.a)) return;
  const size_t e = (size_t)kv_elem_bytes(m.weight_dtype);
  need(aligned(m.q_weight, e) && aligned(m.k_weight, e), "q_weight and k_weight must be aligned to their type");
  if (n.a.q_heads) {
    const Pieces out = pieces(p.q_out, p.q_out_row, p.q_out_head, r.rows, p.q_heads, c.head_dim, (size_t)kv_elem_bytes(c.dtype));
    auto clear = [&](const void* at, uint64_t head, uint32_t heads) {
      return !at || !meet(pieces(at, 0, head, 1, heads, c.head_dim, e), out);
    };
    need(clear(m.q_weight, m.q_weight_head, p.q_heads) && clear(m.k_weight, m.k_weight_head, c.kv_heads),
         "q_out overlaps q_weight or k_weight");
  }
  n.q_weight = static_cast<const char*>(m.q_weight);
  n.k_weight = static_cast<const char*>(m.k_weight);
  n.qw_head = (int64_t)m.q_weight_head;
  n.kw_head = (int64_t)m.k_weight_head;
  n.f32_weight = m.weight_dtype == MIT2CFM_DTYPE_F32;
  n.centered = m.centered != 0;
  n.eps = m.eps;
  const int D = (int)c.head_dim;
  if (c.dtype == MIT2CFM_DTYPE_F32)
    launch<float>(n, D, s);
  else if (c.dtype == MIT2CFM_DTYPE_F16)
    launch<half_t>(n, D, s);
  else
    launch<bf16_t>(n, D, s);
}

}  // namespace mit2hip
