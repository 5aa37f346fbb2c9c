// kv_ops.hip -- operators over a paged key/value cache (see kv_ops.h and
// mit2cfm.h for what they compute).
#include "kv_ops.h"

#include <cmath>
#include <stdexcept>
#include <string>

#include "device_common.h"
#include "engine.h"

namespace mit2hip {

namespace {

typedef __bf16 bf16_t;

void need(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}
void launched(hipError_t e) {
  if (e != hipSuccess) throw HipError(std::string("kv operator launch: ") + hipGetErrorString(e));
}
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// What the kernels take of a cache and of its new rows.
struct CacheView {
  char* k;
  char* v;
  const int32_t* table;
  int pages, page_shift, kv_heads, table_stride;

  // Page that holds a sequence's cached row j (0 <= j < capacity()), or -1.
  __device__ int page_of(int seq, int j) const {
    const int p = table[(size_t)seq * table_stride + (j >> page_shift)];
    return (unsigned)p < (unsigned)pages ? p : -1;
  }
  __device__ int capacity() const { return table_stride << page_shift; }
  // Element index of head 0's row j in a page.
  __device__ int64_t row_in(int page, int j, int D) const {
    return ((((int64_t)page * kv_heads) << page_shift) + (j & ((1 << page_shift) - 1))) * D;
  }
  __device__ int64_t head_stride(int D) const { return (int64_t)D << page_shift; }
};
struct RowView {
  const int32_t* start;
  const int32_t* length;
  int seqs, rows;
};

CacheView view(const mit2cfm_kv_cache& c) {
  return {static_cast<char*>(c.k), static_cast<char*>(c.v), c.table, (int)c.pages,
          __builtin_ctz(c.page_rows), (int)c.kv_heads, (int)c.table_stride};
}
RowView view(const mit2cfm_kv_rows& r) { return {r.start, r.length, (int)r.seqs, (int)r.rows}; }

// The sequence that new row `row` belongs to, or -1 (a wave's lanes look at 64
// bounds at a time; all return the same).
__device__ __forceinline__ int seq_of_row(const RowView& r, int row) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int base = 0; base < r.seqs; base += 64) {
    const bool before = base + lane < r.seqs && r.start[base + lane + 1] <= row;
    const int c = __popcll(__ballot(before));
    n += c;
    if (c < 64) break;
  }
  return n < r.seqs && row >= r.start[n] ? n : -1;
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// ------------------------------------------------------------------ append
constexpr int kAppendThreads = 256;
constexpr int kMaxPairs = 128;  // rotated pairs of a head

struct AppendArgs {
  CacheView c;
  RowView r;
  const char *k, *v, *q;
  char* q_out;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head, qo_row, qo_head;
  const int32_t* position;
  int q_heads, rot, interleaved;
  double log2_theta;
};

// A block takes R rows' items (blockIdx.y: its share of them).  An item is two
// vectors of VEC elements of a head, chosen so that a rotated pair's two
// elements are both in it: (i, i + rot/2), or neighbours when interleaved and
// past the rotated part.  The rows' angles go through LDS once for all heads:
// the angle in turns, fp64, brought to [-1/2, 1/2] there, and its cosine and
// sine in fp32, as everything that follows.
template <typename T, int VEC, int R>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendArgs a, int D) {
  __shared__ float2 turn[R][kMaxPairs];
  __shared__ int64_t s_at[R];  // element index of the row in its page, head 0; -1: not written
  __shared__ int s_place[R];   // the row's position; INT_MIN: no sequence's row
  const int tid = threadIdx.x, row0 = blockIdx.x * R;
  const int wave = tid >> 6;
  for (int i = wave; i < R; i += kAppendThreads / 64) {
    const int row = row0 + i;
    const int seq = row < a.r.rows ? seq_of_row(a.r, row) : -1;
    if ((tid & 63) == 0) {
      int64_t at = -1;
      int pos = INT_MIN;
      if (seq >= 0) {
        const int place = a.r.length[seq] - (a.r.start[seq + 1] - row);
        if (place >= 0 && place < a.c.capacity()) {
          const int page = a.c.page_of(seq, place);
          if (page >= 0) at = a.c.row_in(page, place, D);
        }
        pos = a.position ? a.position[row] : place;
        if (pos == INT_MIN) pos = INT_MIN + 1;
      }
      s_at[i] = at;
      s_place[i] = pos;
    }
  }
  __syncthreads();
  const int half = a.rot >> 1;
  for (int i = tid; i < R * half; i += kAppendThreads) {
    const int rr = i / half, p = i - rr * half;
    const double inv = exp2(-2.0 * p / a.rot * a.log2_theta) * 0.15915494309189533577;  // 1 / (2 pi)
    double t = (double)s_place[rr] * inv;
    t -= rint(t);
    float sn, cs;
    sincospif((float)(2.0 * t), &sn, &cs);
    turn[rr][p] = make_float2(cs, sn);
  }
  __syncthreads();
  const int per_head = D / (2 * VEC);
  const int heads = a.q_heads + 2 * a.c.kv_heads;
  const int items = R * heads * per_head;
  for (int it = blockIdx.y * kAppendThreads + tid; it < items; it += gridDim.y * kAppendThreads) {
    const int u = it % per_head, rh = it / per_head;
    const int h = rh % heads, rr = rh / heads;
    if (s_place[rr] == INT_MIN) continue;
    const int row = row0 + rr;
    // the item's two vectors, and the pair index of its first element
    int e0, e1, pair0;
    const bool rotates = h < a.q_heads + a.c.kv_heads;
    bool turned = false;
    if (a.interleaved || !rotates) {
      e0 = 2 * VEC * u;
      e1 = e0 + VEC;
      pair0 = VEC * u;
      turned = rotates && e0 < a.rot;
    } else if (u * VEC < half) {
      e0 = pair0 = VEC * u;
      e1 = e0 + half;
      turned = true;
    } else {
      e0 = a.rot + 2 * (VEC * u - half);
      e1 = e0 + VEC;
      pair0 = 0;
    }
    const T* src;
    T* dst;
    if (h < a.q_heads) {
      src = reinterpret_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
      dst = reinterpret_cast<T*>(a.q_out) + row * a.qo_row + h * a.qo_head;
    } else {
      if (s_at[rr] < 0) continue;
      const int kh = h - a.q_heads;
      const bool is_k = kh < a.c.kv_heads;
      const int hh = is_k ? kh : kh - a.c.kv_heads;
      src = is_k ? reinterpret_cast<const T*>(a.k) + row * a.k_row + hh * a.k_head
                 : reinterpret_cast<const T*>(a.v) + row * a.v_row + hh * a.v_head;
      dst = reinterpret_cast<T*>(is_k ? a.c.k : a.c.v) + s_at[rr] + hh * a.c.head_stride(D);
    }
    Vec<T, VEC> x = *reinterpret_cast<const Vec<T, VEC>*>(src + e0);
    Vec<T, VEC> y = *reinterpret_cast<const Vec<T, VEC>*>(src + e1);
    if (turned) {
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          // pair j of the item: elements 2 j, 2 j + 1 of (x, y)
          T& p = 2 * j < VEC ? x.v[(2 * j) % VEC] : y.v[(2 * j) % VEC];
          T& q = 2 * j + 1 < VEC ? x.v[(2 * j + 1) % VEC] : y.v[(2 * j + 1) % VEC];
          if (pair0 + j < half) {
            const float2 cs = turn[rr][pair0 + j];
            const float fp = (float)p, fq = (float)q;
            p = (T)(fp * cs.x - fq * cs.y);
            q = (T)(fq * cs.x + fp * cs.y);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 cs = turn[rr][pair0 + j];
          const float fp = (float)x.v[j], fq = (float)y.v[j];
          x.v[j] = (T)(fp * cs.x - fq * cs.y);
          y.v[j] = (T)(fq * cs.x + fp * cs.y);
        }
      }
    }
    *reinterpret_cast<Vec<T, VEC>*>(dst + e0) = x;
    *reinterpret_cast<Vec<T, VEC>*>(dst + e1) = y;
  }
}

template <typename T, int VEC, int R>
void launch_append_rows(const AppendArgs& a, int D, hipStream_t s) {
  const int bx = (a.r.rows + R - 1) / R;
  const int items = R * (a.q_heads + 2 * a.c.kv_heads) * (D / (2 * VEC));
  // few rows: their heads over more blocks, down to one item a thread
  const int by = std::max(1, std::min((items + kAppendThreads - 1) / kAppendThreads, 2048 / bx));
  hipLaunchKernelGGL((append_kernel<T, VEC, R>), dim3(bx, by), dim3(kAppendThreads), 0, s, a, D);
  launched(hipGetLastError());
}

template <typename T>
void launch_append(const AppendArgs& a, int D, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](const void* p, int64_t row, int64_t head) { return aligned(p, 16) && row % V == 0 && head % V == 0; };
  const bool wide = fits(a.k, a.k_row, a.k_head) && fits(a.v, a.v_row, a.v_head) &&
                    (!a.q_heads || (fits(a.q, a.q_row, a.q_head) && fits(a.q_out, a.qo_row, a.qo_head))) &&
                    (a.interleaved || a.rot % (2 * V) == 0);
  // Rows that fill the chip by themselves share a block's angles four at a time.
  if (!wide)
    launch_append_rows<T, 1, 1>(a, D, s);
  else if (a.r.rows >= 2048)
    launch_append_rows<T, V, 4>(a, D, s);
  else
    launch_append_rows<T, V, 1>(a, D, s);
}

// ------------------------------------------------------------------ attention
struct AttendArgs {
  CacheView c;
  RowView r;
  const char* q;
  char* out;
  int64_t q_row, q_head, o_row, o_head;
  const uint32_t* mask;
  int mask_words, q_heads, group, q_wide;
  float scale;
};

// Whether a sequence's new row i sees cached row j; first: its cached rows
// before the new ones.
__device__ __forceinline__ bool sees(const AttendArgs& a, int row, int i, int j, int first) {
  const int n = j - first;
  if (n < 0) return true;
  if (!a.mask) return n <= i;
  return (n >> 5) < a.mask_words && (a.mask[(size_t)row * a.mask_words + (n >> 5)] >> (n & 31) & 1u);
}

// The matrix instruction of a type: its operand, the keys of a tile (KT), and
// the vectors of it that a lane holds for 16 keys and D elements.
template <typename T>
struct Mat;
template <>
struct Mat<half_t> {
  typedef half8 op;
  static constexpr int KT = 32;
  static __device__ __forceinline__ floatx4 mul(const op& a, const op& b, const floatx4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
typedef bf16_t bf8 __attribute__((ext_vector_type(8)));
template <>
struct Mat<bf16_t> {
  typedef bf8 op;
  static constexpr int KT = 32;
  static __device__ __forceinline__ floatx4 mul(const op& a, const op& b, const floatx4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mat<float> {
  typedef float op;
  static constexpr int KT = 16;
  static __device__ __forceinline__ floatx4 mul(const op& a, const op& b, const floatx4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  }
};

template <typename T>
__device__ __forceinline__ bool finite(T v) {
  return fabsf((float)v) < INFINITY;  // (NaN: false)
}

// N elements of a row as a lane reads them, at the alignment that their place
// gives: a multiple of N elements into a 16-byte aligned row.
template <typename T, int N>
struct alignas(N * sizeof(T) % 16 == 0 ? 16 : N * sizeof(T) % 8 == 0 ? 8 : 4) Piece {
  T v[N];
};

constexpr int kAttendWaves = 4, kAttendThreads = kAttendWaves * 64;
constexpr int kChunkStep = 128;  // a split's keys are a multiple: a tile of the longest kind for every wave

// How one launch of the attention is laid out (kv_attention's host side).
struct AttendPlan {
  int tiles;   // M tiles, an upper bound
  int splits;  // of a sequence's keys, at most
  int chunk;   // keys of a split, unless the sequence is longer than splits of them
};

// Keys of a split of a sequence of len keys.
__device__ __forceinline__ int chunk_of(int len, int chunk, int splits) {
  const int least = (len + splits - 1) / splits;
  return max(chunk, (least + kChunkStep - 1) / kChunkStep * kChunkStep);
}

// The sequence and its tile (of `mtile` query rows) that tile number t of the
// whole batch is; false past the last.
__device__ __forceinline__ bool find_tile(const RowView& r, int group, int mtile, int t, int& seq, int& in_seq) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < r.seqs; base += 64) {
    int n = 0;
    if (base + lane < r.seqs) {
      const int s0 = max(r.start[base + lane], 0), s1 = min(r.start[base + lane + 1], r.rows);
      n = s1 > s0 ? (int)(((int64_t)(s1 - s0) * group + mtile - 1) / mtile) : 0;
    }
    int incl = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(incl, off, kWave);
      if (lane >= off) incl += o;
    }
    const uint64_t past = __ballot(before + incl > t);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      seq = base + l;
      in_seq = t - (before + __shfl(incl - n, l, kWave));
      return true;
    }
    before += __shfl(incl, 63, kWave);
  }
  return false;
}

// Attention of 16 MT query rows (a sequence's new rows x the query heads of one
// key head, in that order) over one split of its keys.
//
// Four waves take every fourth tile of KT keys, each with a running softmax,
// and join at the end.  A tile's scores are S^T = K Q^T on the matrix cores: a
// lane ends up with one query (lane % 16) and, of each 16 keys, those from 4 (lane /
// 16) on, which are the slots its group feeds to O^T += V^T P, so the
// probabilities never cross lanes.  K goes straight from memory into the
// operand.  V does too: a lane reads D/16 neighbouring elements of each of its
// keys and turns them into operands by itself, output row i of product d being
// element (D/16) i + d; at the end a lane holds D/4 neighbouring elements of its
// query.  Nothing goes through LDS until the join.
//
// The running maximum is raised only when a score passes it by 2^kSlack (a
// wave-wide vote): up to there the probabilities, at most 2^kSlack, stay exact in
// fp32 sums and in range as 16-bit operands (where they round to the type, as
// the product needs; the sum of the weights keeps fp32).
constexpr float kSlack = 8.f;

template <typename T, int D, int MT, bool BIG>
__global__ __launch_bounds__(kAttendThreads) void attend_kernel(AttendArgs a, AttendPlan plan, float* part_o,
                                                                float2* part_ml) {
  using M = Mat<T>;
  using Op = typename M::op;
  constexpr int KT = M::KT, NT = KT / 16, DP = D / 16;
  constexpr int DC = sizeof(T) == 2 ? D / 32 : D / 4;  // steps of a score's product
  constexpr int NV = KT / 4;                           // a lane's keys of a tile
  constexpr int OS = D + 4;                            // a row of the join's buffer
  __shared__ float sO[kAttendWaves][16][OS];
  __shared__ float2 sML[kAttendWaves][16];
  __shared__ int s_dirty;

  int seq, in_seq;
  if (!find_tile(a.r, a.group, 16 * MT, blockIdx.x, seq, in_seq)) return;
  const int kvh = blockIdx.y, split = blockIdx.z;
  const int start = max(a.r.start[seq], 0), n_all = a.r.start[seq + 1] - a.r.start[seq];
  const int n_new = min(a.r.start[seq + 1], a.r.rows) - start;
  const int first = a.r.length[seq] - n_all, len = min(a.r.length[seq], a.c.capacity());
  const int chunk = chunk_of(max(len, 0), plan.chunk, plan.splits);
  const int begin = split * chunk;
  if (split > 0 && begin >= len) return;
  const int end = min(begin + chunk, len);
  const bool whole = len <= chunk;  // one split: the result is final

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 15, grp = lane >> 4;
  const int mrows = n_new * a.group, m0 = in_seq * 16 * MT;
  if (tid == 0) s_dirty = 0;
  __syncthreads();

  // this lane's queries: their place among the new rows, and the operands
  int qi[MT], qrow[MT];
  Op qv[MT][DC];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int m = min(m0 + 16 * mt + lq, mrows - 1);
    qi[mt] = m / a.group;
    qrow[mt] = start + qi[mt];
    const T* q = reinterpret_cast<const T*>(a.q) + qrow[mt] * a.q_row + (kvh * a.group + (m - qi[mt] * a.group)) * a.q_head;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        if (a.q_wide) {
          qv[mt][c] = *reinterpret_cast<const Op*>(q + 32 * c + 8 * grp);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) qv[mt][c][e] = q[32 * c + 8 * grp + e];
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < DC; ++c) qv[mt][c] = q[D / 4 * grp + c];
    }
    qi[mt] += start - a.r.start[seq];  // (start < 0: rows before the buffer)
  }

  floatx4 o[MT][DP];
  float mx[MT], l[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    mx[mt] = -INFINITY;
    l[mt] = 0.f;
#pragma unroll
    for (int d = 0; d < DP; ++d) o[mt][d] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const float c2 = a.scale * 1.4426950408889634f;  // scores in powers of two
  const int64_t head = kvh * a.c.head_stride(D);
  const T* K = reinterpret_cast<const T*>(a.c.k) + head;
  const T* V = reinterpret_cast<const T*>(a.c.v) + head;
  const int32_t* table = a.c.table + (size_t)seq * a.c.table_stride;
  const int pmask = (1 << a.c.page_shift) - 1;
  const int64_t page_elems = ((int64_t)a.c.kv_heads << a.c.page_shift) * D;
  bool dirty = false;

  // BIG: a tile lies in one page, whose entry is the same for all lanes; else
  // lane i (of the first KT) has key i's entry.
  auto entry = [&](int j0) {
    const int j = BIG ? j0 : j0 + (lane & (KT - 1));
    const int p = table[min(j, len - 1) >> a.c.page_shift];
    return (unsigned)p < (unsigned)a.c.pages && j < len ? p : -1;
  };
  int next = begin + KT * wave < end ? entry(begin + KT * wave) : -1;
  for (int j0 = begin + KT * wave; j0 < end; j0 += KT * kAttendWaves) {
    const int page = next;
    if (j0 + KT * kAttendWaves < end) next = entry(j0 + KT * kAttendWaves);
    if (BIG ? page < 0 : !__any(page >= 0)) continue;
    // operands (rows past the end read the last one's place; they count as unseen)
    Op kv[NT][DC];
    Piece<T, DP> vv[NV];
    uint32_t there;  // bit e: this lane's key e is
    const T *kp[NT], *vp[NV];
    if (BIG) {
      const T* kt = K + page * page_elems;
      const T* vt = V + page * page_elems;
      const int r0 = j0 & pmask, last = min(KT, len - j0) - 1;
#pragma unroll
      for (int t = 0; t < NT; ++t) kp[t] = kt + (r0 + min(16 * t + lq, last)) * D;
      there = 0;
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        const int key = 16 * (e >> 2) + 4 * grp + (e & 3);
        vp[e] = vt + (r0 + min(key, last)) * D;
        there |= (key <= last ? 1u : 0u) << e;
      }
    } else {
      there = 0;
      auto at = [&](int key, const T* base, bool& ok) {
        const int p = __shfl(page, key, kWave);
        ok = p >= 0;
        return base + max(p, 0) * page_elems + ((j0 + key) & pmask) * D;
      };
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        bool ok;
        kp[t] = at(16 * t + lq, K, ok);
      }
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        bool ok;
        vp[e] = at(16 * (e >> 2) + 4 * grp + (e & 3), V, ok);
        there |= (ok ? 1u : 0u) << e;
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int c = 0; c < DC; ++c) kv[t][c] = *reinterpret_cast<const Op*>(kp[t] + 32 * c + 8 * grp);
      } else {
#pragma unroll
        for (int c = 0; c < DC; c += 4) {
          const float4 x = *reinterpret_cast<const float4*>(kp[t] + D / 4 * grp + c);
          kv[t][c] = x.x; kv[t][c + 1] = x.y; kv[t][c + 2] = x.z; kv[t][c + 3] = x.w;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < NV; ++e) vv[e] = *reinterpret_cast<const Piece<T, DP>*>(vp[e] + DP * lq);

    const bool all_there = !__any(there != (1u << NV) - 1u);
    const bool fresh = j0 + KT > first;  // holds new rows, which not every row sees
    if (!all_there) {
#pragma unroll
      for (int e = 0; e < NV; ++e)
        if (!(there >> e & 1u))
#pragma unroll
          for (int d = 0; d < DP; ++d) vv[e].v[d] = (T)0.f;
    }
    if (fresh) {  // 0 x NaN would reach the rows that do not see it: such values join at the end
      bool odd = false;
#pragma unroll
      for (int e = 0; e < NV; ++e)
#pragma unroll
        for (int d = 0; d < DP; ++d)
          if (!finite(vv[e].v[d])) {
            vv[e].v[d] = (T)0.f;
            odd = true;
          }
      dirty = dirty || __any(odd);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float s[NV];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < DC; ++c) acc = M::mul(kv[t][c], qv[mt][c], acc);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * t + r] = acc[r] * c2;
      }
      if (!all_there || fresh) {
        uint32_t seen = there;
        if (fresh) {  // (selects, no branches: every lane forms all its bits)
          const uint32_t* words = a.mask + (size_t)qrow[mt] * a.mask_words;
          uint32_t open = 0;
#pragma unroll
          for (int e = 0; e < NV; ++e) {
            const int n = j0 + 16 * (e >> 2) + 4 * grp + (e & 3) - first;
            uint32_t ok = n <= qi[mt] ? 1u : 0u;
            if (a.mask) {
              const int w = n >> 5;
              ok = words[min(max(w, 0), a.mask_words - 1)] >> (n & 31) & 1u;
              ok = n < 0 ? 1u : w < a.mask_words ? ok : 0u;
            }
            open |= ok << e;
          }
          seen &= open;
        }
#pragma unroll
        for (int e = 0; e < NV; ++e) s[e] = seen >> e & 1u ? s[e] : -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < NV; ++e) top = fmaxf(top, s[e]);
      if (__any(top > mx[mt] + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float mn = fmaxf(mx[mt], top);
        const float alpha = mn == -INFINITY ? 1.f : exp2f(mx[mt] - mn);
        mx[mt] = mn;
        l[mt] *= alpha;
#pragma unroll
        for (int d = 0; d < DP; ++d) o[mt][d] *= alpha;
      }
      const float base = mx[mt] == -INFINITY ? 0.f : mx[mt];
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        s[e] = __builtin_amdgcn_exp2f(s[e] - base);
        l[mt] += s[e];
      }
      if constexpr (sizeof(T) == 2) {
        Op p;
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = (T)s[e];
#pragma unroll
        for (int d = 0; d < DP; ++d) {
          Op v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = vv[e].v[d];
          o[mt][d] = M::mul(v, p, o[mt][d]);
        }
      } else {
#pragma unroll
        for (int d = 0; d < DP; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[mt][d] = M::mul(vv[e].v[d], s[e], o[mt][d]);
      }
    }
  }

  // the join: 16 rows at a time; thread -> row tid / 16, elements DP (tid % 16) ..
  if (dirty && lane == 0) atomicOr(&s_dirty, 1);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float ls = l[mt];
    ls += __shfl_xor(ls, 16, kWave);
    ls += __shfl_xor(ls, 32, kWave);
    if (mt) __syncthreads();
    if (grp == 0) sML[wave][lq] = make_float2(mx[mt], ls);
#pragma unroll
    for (int d = 0; d < DP; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) sO[wave][lq][D / 4 * grp + DP * r + d] = o[mt][d][r];
    __syncthreads();
    const int row16 = tid >> 4, d0 = DP * (tid & 15), m = m0 + 16 * mt + row16;
    if (m < mrows) {
      float mm = sML[0][row16].x;
#pragma unroll
      for (int w = 1; w < kAttendWaves; ++w) mm = fmaxf(mm, sML[w][row16].x);
      const float base = mm == -INFINITY ? 0.f : mm;
      float L = 0.f, O[DP];
#pragma unroll
      for (int d = 0; d < DP; ++d) O[d] = 0.f;
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) {
        const float f = exp2f(sML[w][row16].x - base);
        L += f * sML[w][row16].y;
#pragma unroll
        for (int d = 0; d < DP; ++d) O[d] += f * sO[w][row16][d0 + d];
      }
      const int i = m / a.group, row = start + i, h = kvh * a.group + (m - i * a.group);
      if (s_dirty) {  // new rows' values that are not finite, for the rows that see them
        for (int j = max(begin, max(first, 0)); j < end; ++j) {
          const int p = a.c.page_of(seq, j);
          if (p < 0 || !sees(a, row, i + start - a.r.start[seq], j, first)) continue;
          const T* v = V + p * page_elems + (j & pmask) * D + d0;
          for (int d = 0; d < DP; ++d)
            if (!finite(v[d])) O[d] += (float)v[d];
        }
      }
      if (whole) {
        T* out = reinterpret_cast<T*>(a.out) + row * a.o_row + h * a.o_head + d0;
#pragma unroll
        for (int d = 0; d < DP; ++d) out[d] = (T)(L == 0.f ? 0.f : O[d] / L);
      } else {
        const size_t at = ((size_t)row * a.q_heads + h) * plan.splits + split;
#pragma unroll
        for (int d = 0; d < DP; ++d) part_o[at * D + d0 + d] = O[d];
        if ((tid & 15) == 0) part_ml[at] = make_float2(mm, L);
      }
    }
  }
}

// Joins a row and query head's splits: lane groups of D/4 take every so manyth
// split, four elements a lane.
constexpr int kCombineThreads = 256;
template <typename T, int D>
__global__ __launch_bounds__(kCombineThreads) void combine_kernel(AttendArgs a, AttendPlan plan, const float* part_o,
                                                                  const float2* part_ml) {
  constexpr int L4 = D / 4, G = kCombineThreads / L4;
  __shared__ float4 sO[G][L4];
  __shared__ float sL[G];
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int seq = seq_of_row(a.r, row);
  if (seq < 0) return;
  const int len = min(a.r.length[seq], a.c.capacity());
  const int chunk = chunk_of(max(len, 0), plan.chunk, plan.splits);
  if (len <= chunk) return;
  const int n = (len + chunk - 1) / chunk;
  const size_t at = ((size_t)row * a.q_heads + h) * plan.splits;
  float mm = -INFINITY;
  for (int s = 0; s < n; ++s) mm = fmaxf(mm, part_ml[at + s].x);
  const float base = mm == -INFINITY ? 0.f : mm;
  const int g = tid / L4, l4 = tid - g * L4;
  if (g < G) {
    float L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = g; s < n; s += G) {
      const float2 ml = part_ml[at + s];
      const float f = exp2f(ml.x - base);
      const float4 x = reinterpret_cast<const float4*>(part_o + (at + s) * D)[l4];
      L += f * ml.y;
      O.x += f * x.x; O.y += f * x.y; O.z += f * x.z; O.w += f * x.w;
    }
    sO[g][l4] = O;
    if (l4 == 0) sL[g] = L;
  }
  __syncthreads();
  if (tid >= L4) return;
  float4 O = sO[0][tid];
  float L = sL[0];
#pragma unroll
  for (int w = 1; w < G; ++w) {
    const float4 x = sO[w][tid];
    O.x += x.x; O.y += x.y; O.z += x.z; O.w += x.w;
    L += sL[w];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* out = reinterpret_cast<T*>(a.out) + row * a.o_row + h * a.o_head + 4 * tid;
  const float r[4] = {O.x, O.y, O.z, O.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(L == 0.f ? 0.f : r[e] * inv);
}

// Query rows of a tile for a batch: the average sequence's, up to four matrix
// tiles (at head sizes past 128 two: their accumulators fill the registers).
int m_tiles(uint64_t rows, uint64_t seqs, int group, int D) {
  const uint64_t m = rows * (uint64_t)group / seqs;
  return m <= 16 ? 1 : m <= 32 || D > 128 ? 2 : 4;
}

constexpr int kBlocksWanted = 1024;  // four of these blocks a CU
constexpr int kMaxSplits = 128;

AttendPlan attend_plan(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads) {
  const int group = (int)(q_heads / c.kv_heads);
  const int mtile = 16 * m_tiles(r.rows, r.seqs, group, (int)c.head_dim);
  // sum over the sequences of ceil(rows * group / mtile): at most ...
  const uint64_t by_fill = ((uint64_t)r.rows * group + (uint64_t)std::min(r.seqs, r.rows) * (mtile - 1)) / mtile;
  const uint64_t by_row = (uint64_t)r.rows * ((group + mtile - 1) / mtile);
  AttendPlan p;
  p.tiles = (int)std::min(by_fill, by_row);
  const uint64_t blocks = (uint64_t)p.tiles * c.kv_heads;
  const uint64_t len = std::max<uint64_t>(1, std::min<uint64_t>(r.max_length, (uint64_t)c.table_stride * c.page_rows));
  const uint64_t most = std::min<uint64_t>((len + kChunkStep - 1) / kChunkStep, kMaxSplits);
  const uint64_t splits = std::min<uint64_t>(most, (kBlocksWanted + blocks - 1) / blocks);
  p.chunk = (int)(((len + splits - 1) / splits + kChunkStep - 1) / kChunkStep * kChunkStep);
  p.splits = (int)((len + p.chunk - 1) / p.chunk);
  return p;
}

template <typename T, int D, int MT>
void launch_attend_tile(const AttendArgs& a, const AttendPlan& plan, float* part_o, float2* part_ml, hipStream_t s) {
  const dim3 grid(plan.tiles, a.c.kv_heads, plan.splits), block(kAttendThreads);
  if ((1 << a.c.page_shift) >= Mat<T>::KT)
    hipLaunchKernelGGL((attend_kernel<T, D, MT, true>), grid, block, 0, s, a, plan, part_o, part_ml);
  else
    hipLaunchKernelGGL((attend_kernel<T, D, MT, false>), grid, block, 0, s, a, plan, part_o, part_ml);
  launched(hipGetLastError());
}

template <typename T, int D>
void launch_attend(const AttendArgs& a, const AttendPlan& plan, void* workspace, hipStream_t s) {
  const size_t n = (size_t)a.r.rows * a.q_heads * plan.splits;
  float* part_o = static_cast<float*>(workspace);
  float2* part_ml = reinterpret_cast<float2*>(part_o + n * D);
  const int mt = m_tiles(a.r.rows, a.r.seqs, a.group, D);
  if (mt == 1)
    launch_attend_tile<T, D, 1>(a, plan, part_o, part_ml, s);
  else if (mt == 2)
    launch_attend_tile<T, D, 2>(a, plan, part_o, part_ml, s);
  else if constexpr (D <= 128)
    launch_attend_tile<T, D, 4>(a, plan, part_o, part_ml, s);
  if (plan.splits == 1) return;
  hipLaunchKernelGGL((combine_kernel<T, D>), dim3(a.r.rows, a.q_heads), dim3(kCombineThreads), 0, s, a, plan, part_o,
                     part_ml);
  launched(hipGetLastError());
}

template <typename T>
void launch_attend_dim(const AttendArgs& a, const AttendPlan& plan, int D, void* workspace, hipStream_t s) {
  switch (D) {
    case 32: return launch_attend<T, 32>(a, plan, workspace, s);
    case 64: return launch_attend<T, 64>(a, plan, workspace, s);
    case 96: return launch_attend<T, 96>(a, plan, workspace, s);
    case 128: return launch_attend<T, 128>(a, plan, workspace, s);
    case 192: return launch_attend<T, 192>(a, plan, workspace, s);
    case 256: return launch_attend<T, 256>(a, plan, workspace, s);
  }
}

void check_rows(const mit2cfm_kv_rows& r) {
  need(r.seqs <= 65535, "seqs must be <= 65535");
  need(r.rows < (1u << 24), "rows must be below 2^24");
  need(r.seqs == 0 || r.rows == 0 || (r.start && r.length), "start and length must not be NULL");
}

// An output's rows and heads must not lie on one another.
void check_out(uint64_t row, uint64_t head, uint32_t rows, uint32_t heads, uint32_t D, const char* what) {
  need((heads <= 1 || head >= D) && (rows <= 1 || row >= D), what);
}

}  // namespace

int kv_elem_bytes(int32_t dtype) { return dtype == MIT2CFM_DTYPE_F32 ? 4 : 2; }

void check_kv_cache(const mit2cfm_kv_cache& c) {
  need(c.dtype >= MIT2CFM_DTYPE_F32 && c.dtype <= MIT2CFM_DTYPE_BF16, "the cache's dtype must be f32, f16 or bf16");
  need(c.page_rows >= 1 && c.page_rows <= 1024 && (c.page_rows & (c.page_rows - 1)) == 0,
       "page_rows must be a power of two in [1, 1024]");
  need(c.kv_heads >= 1 && c.kv_heads <= 1024, "kv_heads must be in [1, 1024]");
  need(c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 96 || c.head_dim == 128 || c.head_dim == 192 ||
           c.head_dim == 256,
       "head_dim must be 32, 64, 96, 128, 192 or 256");
  need(c.pages >= 1 && c.pages < (1u << 31), "pages must be in [1, 2^31)");
  need(c.table_stride >= 1 && (uint64_t)c.table_stride * c.page_rows < (1ull << 31),
       "table_stride must be >= 1, page_rows * table_stride below 2^31");
  need(c.k && c.v && c.table, "the cache's k, v and table must not be NULL");
  need(aligned(c.k, 16) && aligned(c.v, 16), "the cache's k and v must be 16-byte aligned");
}

void kv_append(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, const mit2cfm_kv_append& p, hipStream_t s) {
  check_kv_cache(c);
  check_rows(r);
  need(p.q_heads <= 4096, "q_heads must be <= 4096");
  need(p.rotary_dim <= c.head_dim && p.rotary_dim % 2 == 0, "rotary_dim must be even and <= head_dim");
  need(p.rotary_dim == 0 || (p.theta > 0.0 && std::isfinite(p.theta)), "theta must be positive and finite");
  if (r.seqs == 0 || r.rows == 0) return;
  const bool with_q = p.q != nullptr;
  need(p.k && p.v, "k and v must not be NULL");
  need(!with_q || (p.q_out && p.q_heads > 0), "q needs q_out and q_heads");
  const size_t e = (size_t)kv_elem_bytes(c.dtype);
  need(aligned(p.k, e) && aligned(p.v, e) && aligned(p.q, e) && aligned(p.q_out, e),
       "k, v, q and q_out must be aligned to their type");
  if (with_q) {
    check_out(p.q_out_row, p.q_out_head, r.rows, p.q_heads, c.head_dim, "q_out's rows and heads overlap");
    need(p.q != p.q_out || (p.q_row == p.q_out_row && p.q_head == p.q_out_head),
         "q_out may be q only with its strides");
  }
  AppendArgs a;
  a.c = view(c);
  a.r = view(r);
  a.k = static_cast<const char*>(p.k);
  a.v = static_cast<const char*>(p.v);
  a.q = static_cast<const char*>(p.q);
  a.q_out = static_cast<char*>(p.q_out);
  a.k_row = (int64_t)p.k_row; a.k_head = (int64_t)p.k_head;
  a.v_row = (int64_t)p.v_row; a.v_head = (int64_t)p.v_head;
  a.q_row = (int64_t)p.q_row; a.q_head = (int64_t)p.q_head;
  a.qo_row = (int64_t)p.q_out_row; a.qo_head = (int64_t)p.q_out_head;
  a.position = p.position;
  a.q_heads = with_q ? (int)p.q_heads : 0;
  a.rot = (int)p.rotary_dim;
  a.interleaved = p.interleaved != 0;
  a.log2_theta = p.rotary_dim ? std::log2(p.theta) : 0.0;
  const int D = (int)c.head_dim;
  if (c.dtype == MIT2CFM_DTYPE_F32)
    launch_append<float>(a, D, s);
  else if (c.dtype == MIT2CFM_DTYPE_F16)
    launch_append<half_t>(a, D, s);
  else
    launch_append<bf16_t>(a, D, s);
}

uint64_t kv_attention_workspace(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads) {
  if (c.kv_heads < 1 || c.kv_heads > 1024 || c.head_dim < 32 || c.head_dim > 256 || c.page_rows < 1 || c.table_stride < 1 ||
      q_heads < 1 || q_heads > 4096 || q_heads % c.kv_heads || r.seqs < 1 || r.seqs > 65535 || r.rows < 1 ||
      r.rows >= (1u << 24))
    return 0;
  const AttendPlan plan = attend_plan(c, r, q_heads);
  if (plan.splits == 1) return 0;
  return (uint64_t)r.rows * q_heads * plan.splits * (c.head_dim + 2) * sizeof(float);
}

void kv_attention(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, const mit2cfm_kv_attention& p, hipStream_t s) {
  check_kv_cache(c);
  check_rows(r);
  need(p.q_heads >= 1 && p.q_heads <= 4096 && p.q_heads % c.kv_heads == 0,
       "q_heads must be a multiple of kv_heads, <= 4096");
  need(std::isfinite(p.scale), "scale must be finite");
  need(p.mask == nullptr || p.mask_words >= 1, "mask_words must be >= 1 with a mask");
  need(p.mask_words < (1u << 24), "mask_words must be below 2^24");
  if (r.seqs == 0 || r.rows == 0) return;
  need(p.q && p.out, "q and out must not be NULL");
  const size_t e = (size_t)kv_elem_bytes(c.dtype);
  need(aligned(p.q, e) && aligned(p.out, e), "q and out must be aligned to their type");
  check_out(p.out_row, p.out_head, r.rows, p.q_heads, c.head_dim, "out's rows and heads overlap");
  const uint64_t bytes = kv_attention_workspace(c, r, p.q_heads);
  need(bytes == 0 || (p.workspace && p.workspace_bytes >= bytes), "workspace is NULL or too small");
  need(aligned(p.workspace, 16), "workspace must be 16-byte aligned");
  AttendArgs a;
  a.c = view(c);
  a.r = view(r);
  a.q = static_cast<const char*>(p.q);
  a.out = static_cast<char*>(p.out);
  a.q_row = (int64_t)p.q_row; a.q_head = (int64_t)p.q_head;
  a.o_row = (int64_t)p.out_row; a.o_head = (int64_t)p.out_head;
  a.mask = p.mask;
  a.mask_words = p.mask ? (int)p.mask_words : 0;
  a.q_heads = (int)p.q_heads;
  a.group = (int)(p.q_heads / c.kv_heads);
  a.scale = p.scale;
  a.q_wide = aligned(p.q, 16) && p.q_row % 8 == 0 && p.q_head % 8 == 0;
  const int D = (int)c.head_dim;
  const AttendPlan plan = attend_plan(c, r, p.q_heads);
  if (c.dtype == MIT2CFM_DTYPE_F32)
    launch_attend_dim<float>(a, plan, D, p.workspace, s);
  else if (c.dtype == MIT2CFM_DTYPE_F16)
    launch_attend_dim<half_t>(a, plan, D, p.workspace, s);
  else
    launch_attend_dim<bf16_t>(a, plan, D, p.workspace, s);
}

}  // namespace mit2hip
