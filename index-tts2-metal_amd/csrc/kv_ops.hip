// kv_ops.hip -- operators over a paged key/value cache (see kv_ops.h and
// mit2cfm.h for what they compute).
#include "kv_ops.h"

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "engine.h"
#include "kv_attend.h"
#include "kv_view.h"
#include "overlap.h"

namespace mit2hip {

namespace {

void need(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}
void launched(hipError_t e) {
  if (e != hipSuccess) throw HipError(std::string("kv operator launch: ") + hipGetErrorString(e));
}
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

CacheView view(const mit2cfm_kv_cache& c) {
  return {static_cast<char*>(c.k), static_cast<char*>(c.v), c.table, (int)c.pages,
          __builtin_ctz(c.page_rows), (int)c.kv_heads, (int)c.table_stride};
}
RowView view(const mit2cfm_kv_rows& r) { return {r.start, r.length, (int)r.seqs, (int)r.rows}; }

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

// A block takes a row's items (blockIdx.y: its share of them).  An item is two
// vectors of VEC elements of a head, chosen so that a rotated pair's two
// elements are both in it: (i, i + rot/2), or neighbours when interleaved and
// past the rotated part.  The row's angles go through LDS once for all heads:
// the angle in turns, fp64, brought to [-1/2, 1/2] there, and its cosine and
// sine in fp32, as everything that follows.  The result's rounding to the type is
// the only one to fewer bits.
//
// Bound by its reads and writes: nine prompts of up to 2047 rows, 32 + 2 x 8 heads of
// 128 bf16, 332 MB in 64 us (5.2 TB/s; a large copy reaches 4.7), four rows a block in
// 69.  Trees of 25 rows of 16 sequences take 4.5 us and three single rows 2.8, mostly
// the launch and two waits in a row (the row's sequence, then its page).
template <typename T, int VEC>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendArgs a, int D) {
  __shared__ float2 turn[kMaxPairs];
  __shared__ int64_t s_at;  // element index of the row in its page, head 0; -1: not written
  __shared__ int s_place;   // the row's position
  __shared__ int s_mine;    // the row is a sequence's
  const int tid = threadIdx.x, row = blockIdx.x;
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
  }
  __syncthreads();
  if (!s_mine) return;
  const int half = a.rot >> 1;
  for (int p = tid; p < half; p += kAppendThreads) {
    const double inv = exp2(-2.0 * p / a.rot * a.log2_theta) * 0.15915494309189533577;  // 1 / (2 pi)
    double t = (double)s_place * inv;
    t -= rint(t);
    float sn, cs;
    sincospif((float)(2.0 * t), &sn, &cs);
    turn[p] = make_float2(cs, sn);
  }
  __syncthreads();
  const int per_head = D / (2 * VEC);
  const int items = (a.q_heads + 2 * a.c.kv_heads) * per_head;
  for (int it = blockIdx.y * kAppendThreads + tid; it < items; it += gridDim.y * kAppendThreads) {
    const int u = it % per_head, h = it / per_head;
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
      if (s_at < 0) continue;
      const int kh = h - a.q_heads;
      const bool is_k = kh < a.c.kv_heads;
      const int hh = is_k ? kh : kh - a.c.kv_heads;
      src = is_k ? reinterpret_cast<const T*>(a.k) + row * a.k_row + hh * a.k_head
                 : reinterpret_cast<const T*>(a.v) + row * a.v_row + hh * a.v_head;
      dst = reinterpret_cast<T*>(is_k ? a.c.k : a.c.v) + s_at + hh * a.c.head_stride(D);
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
            const float2 cs = turn[pair0 + j];
            const float fp = (float)p, fq = (float)q;
            p = (T)(fp * cs.x - fq * cs.y);
            q = (T)(fq * cs.x + fp * cs.y);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 cs = turn[pair0 + j];
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

template <typename T, int VEC>
void launch_append_by(const AppendArgs& a, int D, hipStream_t s) {
  const int items = (a.q_heads + 2 * a.c.kv_heads) * (D / (2 * VEC));
  // few rows: their heads over more blocks, down to one item a thread
  const int by = std::max(1, std::min((items + kAppendThreads - 1) / kAppendThreads, 2048 / a.r.rows));
  hipLaunchKernelGGL((append_kernel<T, VEC>), dim3(a.r.rows, by), dim3(kAppendThreads), 0, s, a, D);
  launched(hipGetLastError());
}

template <typename T>
void launch_append(const AppendArgs& a, int D, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](const void* p, int64_t row, int64_t head) { return aligned(p, 16) && row % V == 0 && head % V == 0; };
  const bool wide = fits(a.k, a.k_row, a.k_head) && fits(a.v, a.v_row, a.v_head) &&
                    (!a.q_heads || (fits(a.q, a.q_row, a.q_head) && fits(a.q_out, a.qo_row, a.qo_head))) &&
                    (a.interleaved || a.rot % (2 * V) == 0);
  if (wide)
    launch_append_by<T, V>(a, D, s);
  else
    launch_append_by<T, 1>(a, D, s);
}

// ------------------------------------------------------------------ attention
void check_rows(const mit2cfm_kv_rows& r) {
  need(r.seqs <= 65535, "seqs must be <= 65535");
  need(r.rows < (1u << 24), "rows must be below 2^24");
  need(r.seqs == 0 || r.rows == 0 || (r.start && r.length), "start and length must not be NULL");
  need(aligned(r.start, 4) && aligned(r.length, 4), "start and length must be 4-byte aligned");
}

// What attend_plan's numbers, and the kernels' 32-bit ones of query rows, are made for.
bool attention_in_range(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, uint32_t q_heads) {
  return q_heads >= 1 && q_heads <= 4096 && q_heads % c.kv_heads == 0 && (uint64_t)r.rows * q_heads <= (1u << 28);
}

}  // namespace

void attend_launched(hipError_t e) { launched(e); }

int kv_elem_bytes(int32_t dtype) { return dtype == MIT2CFM_DTYPE_F32 ? 4 : 2; }

namespace {
void check_kv_sizes(const mit2cfm_kv_cache& c) {
  need(c.dtype >= MIT2CFM_DTYPE_F32 && c.dtype <= MIT2CFM_DTYPE_BF16, "the cache's dtype must be f32, f16 or bf16");
  need(c.page_rows >= 1 && c.page_rows <= 1024 && (c.page_rows & (c.page_rows - 1)) == 0,
       "page_rows must be a power of two in [1, 1024]");
  need(c.kv_heads >= 1 && c.kv_heads <= 1024, "kv_heads must be in [1, 1024]");
  need(c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 96 || c.head_dim == 128 || c.head_dim == 192 ||
           c.head_dim == 256,
       "head_dim must be 32, 64, 96, 128, 192 or 256");
  need(c.pages >= 1 && c.pages < (1u << 31), "pages must be in [1, 2^31)");
  need(c.table_stride >= 1 && (uint64_t)c.table_stride * c.page_rows <= (1u << 30),
       "table_stride must be >= 1, page_rows * table_stride <= 2^30");
}
}  // namespace

void check_kv_cache(const mit2cfm_kv_cache& c) {
  check_kv_sizes(c);
  need(c.k && c.v && c.table, "the cache's k, v and table must not be NULL");
  need(aligned(c.k, 16) && aligned(c.v, 16) && aligned(c.table, 4),
       "the cache's k and v must be 16-byte aligned, its table 4-byte aligned");
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
  need(aligned(p.position, 4), "position must be 4-byte aligned");
  if (with_q) {
    auto set = [&](const void* at, uint64_t row, uint64_t head, uint32_t heads) {
      return pieces(at, row, head, r.rows, heads, c.head_dim, e);
    };
    const Pieces out = set(p.q_out, p.q_out_row, p.q_out_head, p.q_heads);
    need(!meet_themselves(out), "q_out's rows and heads overlap");
    need(p.q != p.q_out || (p.q_row == p.q_out_row && p.q_head == p.q_out_head),
         "q_out may be q only with its strides");
    need(p.q == p.q_out || !meet(set(p.q, p.q_row, p.q_head, p.q_heads), out), "q_out overlaps q");
    need(!meet(set(p.k, p.k_row, p.k_head, c.kv_heads), out) && !meet(set(p.v, p.v_row, p.v_head, c.kv_heads), out),
         "q_out overlaps k or v");
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
  try {
    check_kv_sizes(c);
    check_rows(r);
  } catch (const std::invalid_argument&) {
    return 0;
  }
  if (r.seqs == 0 || r.rows == 0 || !attention_in_range(c, r, q_heads)) return 0;
  const AttendPlan plan = attend_plan(c, r, q_heads);
  if (plan.splits == 1) return 0;
  return (uint64_t)r.rows * q_heads * (plan.splits * (uint64_t)(c.head_dim + 2) + 1) * sizeof(float);
}

void kv_attention(const mit2cfm_kv_cache& c, const mit2cfm_kv_rows& r, const mit2cfm_kv_attention& p, hipStream_t s) {
  check_kv_cache(c);
  check_rows(r);
  need(attention_in_range(c, r, p.q_heads),
       "q_heads must be a multiple of kv_heads, <= 4096, rows * q_heads <= 2^28");
  need(std::isfinite(p.scale), "scale must be finite");
  need(p.mask == nullptr || p.mask_words >= 1, "mask_words must be >= 1 with a mask");
  need(p.mask_words < (1u << 24), "mask_words must be below 2^24");
  need(aligned(p.mask, 4), "mask must be 4-byte aligned");
  if (r.seqs == 0 || r.rows == 0) return;
  need(p.q && p.out && p.q != p.out, "q and out must not be NULL, nor the same");
  const size_t e = (size_t)kv_elem_bytes(c.dtype);
  need(aligned(p.q, e) && aligned(p.out, e), "q and out must be aligned to their type");
  const Pieces out = pieces(p.out, p.out_row, p.out_head, r.rows, p.q_heads, c.head_dim, e);
  need(!meet_themselves(out), "out's rows and heads overlap");
  need(!meet(pieces(p.q, p.q_row, p.q_head, r.rows, p.q_heads, c.head_dim, e), out), "out overlaps q");
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
  a.flip = p.scale < 0.f;
  a.scale2 = std::max(std::fabs(p.scale) * 1.4426950408889634f, 1e-37f);  // (0: masked scores stay -inf)
  a.q_wide = aligned(p.q, 16) && p.q_row % 8 == 0 && p.q_head % 8 == 0;
  a.o_wide = aligned(p.out, 16) && p.out_row % 8 == 0 && p.out_head % 8 == 0;
  const int D = (int)c.head_dim;
  const AttendPlan plan = attend_plan(c, r, p.q_heads);
  if (c.dtype == MIT2CFM_DTYPE_F32)
    launch_attend_f32(a, plan, D, p.workspace, s);
  else if (c.dtype == MIT2CFM_DTYPE_F16)
    launch_attend_f16(a, plan, D, p.workspace, s);
  else
    launch_attend_bf16(a, plan, D, p.workspace, s);
}

}  // namespace mit2hip
