// beam_ops.hip -- a beam search's step (see beam_ops.h and mit2cfm.h for what
// the operators compute).
#include "beam_ops.h"

#include <cfloat>
#include <stdexcept>
#include <string>

#include "device_common.h"
#include "engine.h"
#include "kv_ops.h"

namespace mit2hip {

namespace {

typedef __bf16 bf16_t;

void need(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}
void launched(hipError_t e) {
  if (e != hipSuccess) throw HipError(std::string("beam operator launch: ") + hipGetErrorString(e));
}
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

constexpr int kMaxBeams = 64, kMaxCount = 64;

// ------------------------------------------------------------------ select
struct SelectArgs {
  const void* logits;
  int64_t row;
  int groups, beams, vocab, count, stop;
  const float* scores;
  const int32_t* finished;
  float* scores_out;
  int32_t *parent_out, *token_out, *finished_out;
  double* sums;   // workspace: [rows] sum of exp(x - max)
  float* tops;    // [rows] max
  float* cand_x;  // [rows][count] the row's best logits, in order
  int32_t* cand_t;
};

constexpr int kSelectThreads = 256;

// A logit as the selection sees it.
template <typename T>
__device__ __forceinline__ float logit(T v) {
  const float x = (float)v;
  return x != x ? -INFINITY : fminf(x, FLT_MAX);
}

struct Best {
  float x;
  int t;
};
__device__ __forceinline__ bool better(float ax, int at, float bx, int bt) { return ax > bx || (ax == bx && at < bt); }

// Block (row): its maximum, the sum of its exponentials, its `count` best.
template <typename T>
__global__ __launch_bounds__(kSelectThreads) void select_rows_kernel(SelectArgs a) {
  __shared__ float sx[kSelectThreads / 64];
  __shared__ int stt[kSelectThreads / 64];
  __shared__ double ss[kSelectThreads / 64];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* x = static_cast<const T*>(a.logits) + r * a.row;
  float px = INFINITY;
  int pt = -1;
  float m = -INFINITY;
  for (int k = 0; k < a.count && k < a.vocab; ++k) {
    float bx = -INFINITY;
    int bt = INT_MAX;
    for (int t = tid; t < a.vocab; t += kSelectThreads) {
      const float v = logit(x[t]);
      if ((v < px || (v == px && t > pt)) && better(v, t, bx, bt)) {
        bx = v;
        bt = t;
      }
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) {
      const float ox = __shfl_xor(bx, off, kWave);
      const int ot = __shfl_xor(bt, off, kWave);
      if (better(ox, ot, bx, bt)) {
        bx = ox;
        bt = ot;
      }
    }
    __syncthreads();
    if (lane == 0) {
      sx[wave] = bx;
      stt[wave] = bt;
    }
    __syncthreads();
    for (int w = 0; w < kSelectThreads / 64; ++w)
      if (w == 0 || better(sx[w], stt[w], bx, bt)) {
        bx = sx[w];
        bt = stt[w];
      }
    if (k == 0) m = bx;
    px = bx;
    pt = bt;
    if (tid == 0) {
      a.cand_x[(size_t)r * a.count + k] = bx;
      a.cand_t[(size_t)r * a.count + k] = bt;
    }
  }
  double sum = 0.0;
  const float ms = m == -INFINITY ? 0.f : m;
  for (int t = tid; t < a.vocab; t += kSelectThreads) sum += (double)expf(logit(x[t]) - ms);
#pragma unroll
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, kWave);
  if (lane == 0) ss[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kSelectThreads / 64; ++w) sum += ss[w];
    a.sums[r] = sum;
    a.tops[r] = m;
  }
}

// Block (group): the best of its beams' candidates.
__global__ __launch_bounds__(kSelectThreads) void select_group_kernel(SelectArgs a) {
  __shared__ double sv[kMaxBeams * kMaxCount];
  __shared__ int stt[kMaxBeams * kMaxCount];
  const int g = blockIdx.x, tid = threadIdx.x, n = a.beams * min(a.count, a.vocab);
  const int per = min(a.count, a.vocab);
  for (int c = tid; c < n; c += kSelectThreads) {
    const int b = c / per, k = c - b * per, r = g * a.beams + b;
    const float cum = a.scores[r];
    const bool done = a.finished && a.finished[r] != 0;
    double s = -INFINITY;
    int t = k;
    if (!(cum > -INFINITY)) {
      // no such beam: the lowest tokens, at -inf
    } else if (done) {  // the stop token, then the lowest others at -inf
      t = k == 0 ? a.stop : (k - 1 < a.stop ? k - 1 : k);
      s = k == 0 ? (double)cum : -INFINITY;
    } else {
      const float x = a.cand_x[(size_t)r * a.count + k];
      t = a.cand_t[(size_t)r * a.count + k];
      if (x > -INFINITY) s = (double)cum + ((double)x - ((double)a.tops[r] + log(a.sums[r])));
    }
    sv[c] = s;
    stt[c] = t;
  }
  __syncthreads();
  for (int c = tid; c < n; c += kSelectThreads) {
    const int b = c / per, t = stt[c];
    const double s = sv[c];
    int rank = 0;
    for (int o = 0; o < n; ++o) {
      const double os = sv[o];
      const int ob = o / per;
      rank += os > s || (os == s && (ob < b || (ob == b && stt[o] < t)));
    }
    if (rank >= a.count) continue;
    const size_t at = (size_t)g * a.count + rank;
    a.scores_out[at] = (float)s;
    a.parent_out[at] = b;
    a.token_out[at] = t;
    if (a.finished_out)
      a.finished_out[at] = t == a.stop || (a.finished && a.finished[g * a.beams + b] != 0) ? 1 : 0;
  }
}

bool select_in_range(const mit2cfm_beam_select& a) {
  return a.dtype >= MIT2CFM_DTYPE_F32 && a.dtype <= MIT2CFM_DTYPE_BF16 && a.beams >= 1 && a.beams <= (uint32_t)kMaxBeams &&
         a.vocab >= 1 && a.vocab <= (1u << 24) && a.count >= 1 && a.count <= (uint32_t)kMaxCount &&
         a.count <= (uint64_t)a.beams * a.vocab && (uint64_t)a.groups * a.beams <= (1u << 20);
}
size_t align16(size_t b) { return (b + 15) & ~size_t(15); }

// ------------------------------------------------------------------ reorder
struct ReorderArgs {
  char *k, *v;
  const int32_t* table;
  int32_t* table_out;
  int pages, page_shift, kv_heads, table_stride;
  int beams;
  int row16;              // 16-byte vectors of a cached row
  int64_t layer16;        //   and from a layer to the next
  const int32_t* parent;
  int64_t parent_stride;
  const int32_t* length;
  const uint32_t* state;
  uint32_t* state_out;
  int state_words;
  const uint32_t* token;
  const int32_t* place;
};

constexpr int kReorderThreads = 256;

// Block (new beam, part): part 0 writes the beam's table row and states, part 1
// + 2 l (+ 1) copies the part page's k (v) of layer l, for a beam that is not
// its parent's first child.  Each block finds whose pages are whose by itself,
// from the group's parents as bits: a beam is a further child when an earlier
// one has its parent, its rank among those is its index less the distinct
// parents before it, and there are as many beams without children.
__global__ __launch_bounds__(kReorderThreads) void reorder_kernel(ReorderArgs a) {
  const int r = blockIdx.x, g = r / a.beams, b = r - g * a.beams;
  const int tid = threadIdx.x, lane = tid & 63;
  int p = lane;
  if (lane < a.beams) {
    const int given = a.parent[g * a.parent_stride + lane];
    if ((unsigned)given < (unsigned)a.beams) p = given;
  }
  uint64_t all = lane < a.beams ? 1ull << p : 0ull, before = lane < b ? 1ull << p : 0ull;
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    all |= __shfl_xor((unsigned long long)all, off, kWave);
    before |= __shfl_xor((unsigned long long)before, off, kWave);
  }
  const int mine = __shfl(p, b, kWave);
  const bool further = (before >> mine) & 1ull;
  int owner = mine;
  if (further) {
    uint64_t bare = ~all & (a.beams == 64 ? ~0ull : (1ull << a.beams) - 1ull);
    for (int k = b - __popcll(before); k > 0; --k) bare &= bare - 1;
    owner = __ffsll((unsigned long long)bare) - 1;
  }
  int len = a.length[g];
  const int capacity = a.table_stride << a.page_shift;
  if (len < 0 || len > capacity) len = capacity;
  const int full = len >> a.page_shift, part = len & ((1 << a.page_shift) - 1);
  const int32_t* from = a.table + ((size_t)g * a.beams + mine) * a.table_stride;
  const int32_t* priv = a.table + ((size_t)g * a.beams + owner) * a.table_stride;
  if (blockIdx.y == 0) {
    int32_t* to = a.table_out + (size_t)r * a.table_stride;
    for (int j = tid; j < a.table_stride; j += kReorderThreads) to[j] = j < full ? from[j] : priv[j];
    if (a.state) {
      const uint32_t* src = a.state + ((size_t)g * a.beams + mine) * a.state_words;
      uint32_t* dst = a.state_out + (size_t)r * a.state_words;
      const int at = a.token ? a.place[g] : -1;
      for (int j = tid; j < a.state_words; j += kReorderThreads)
        dst[j] = j == at ? a.token[g * a.parent_stride + b] : src[j];
    }
    return;
  }
  if (!further || part == 0) return;
  const int src = from[full], dst = priv[full];
  if ((unsigned)src >= (unsigned)a.pages || (unsigned)dst >= (unsigned)a.pages) return;
  const int y = blockIdx.y - 1;
  uint4* base = reinterpret_cast<uint4*>(y & 1 ? a.v : a.k) + (y >> 1) * a.layer16;
  const int per = part * a.row16;  // a head's vectors
  const int64_t head = (int64_t)a.row16 << a.page_shift;
  const uint4* s = base + (int64_t)src * a.kv_heads * head;
  uint4* d = base + (int64_t)dst * a.kv_heads * head;
  for (int i = tid; i < per * a.kv_heads; i += kReorderThreads) {
    const int h = i / per, e = i - h * per;
    d[h * head + e] = s[h * head + e];
  }
}

}  // namespace

uint64_t beam_select_workspace(const mit2cfm_beam_select& a) {
  if (!select_in_range(a)) return 0;
  const size_t rows = (size_t)a.groups * a.beams;
  return align16(rows * 8) + align16(rows * 4) + 2 * align16(rows * a.count * 4) + 16;
}

void beam_select(const mit2cfm_beam_select& p, hipStream_t s) {
  need(select_in_range(p), "dtype, beams, vocab, count or groups * beams out of range");
  need(p.stop_token >= -1 && (p.stop_token < 0 || (uint32_t)p.stop_token < p.vocab), "stop_token must be -1 or in [0, vocab)");
  need(p.finished == nullptr || p.stop_token >= 0, "finished needs a stop_token");
  if (p.groups == 0) return;
  need(p.logits && p.scores && p.scores_out && p.parent_out && p.token_out,
       "logits, scores, scores_out, parent_out and token_out must not be NULL");
  need(aligned(p.logits, (size_t)kv_elem_bytes(p.dtype)), "logits must be aligned to its type");
  need(p.workspace && p.workspace_bytes >= beam_select_workspace(p), "workspace is NULL or too small");
  need(aligned(p.workspace, 16), "workspace must be 16-byte aligned");
  const size_t rows = (size_t)p.groups * p.beams;
  SelectArgs a;
  a.logits = p.logits;
  a.row = (int64_t)p.logits_row;
  a.groups = (int)p.groups; a.beams = (int)p.beams; a.vocab = (int)p.vocab; a.count = (int)p.count;
  a.stop = p.stop_token;
  a.scores = p.scores; a.finished = p.finished;
  a.scores_out = p.scores_out; a.parent_out = p.parent_out; a.token_out = p.token_out; a.finished_out = p.finished_out;
  char* w = static_cast<char*>(p.workspace);
  a.sums = reinterpret_cast<double*>(w);
  w += align16(rows * 8);
  a.tops = reinterpret_cast<float*>(w);
  w += align16(rows * 4);
  a.cand_x = reinterpret_cast<float*>(w);
  w += align16(rows * a.count * 4);
  a.cand_t = reinterpret_cast<int32_t*>(w);
  const dim3 grid((uint32_t)rows), block(kSelectThreads);
  if (p.dtype == MIT2CFM_DTYPE_F32)
    hipLaunchKernelGGL((select_rows_kernel<float>), grid, block, 0, s, a);
  else if (p.dtype == MIT2CFM_DTYPE_F16)
    hipLaunchKernelGGL((select_rows_kernel<half_t>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((select_rows_kernel<bf16_t>), grid, block, 0, s, a);
  launched(hipGetLastError());
  hipLaunchKernelGGL(select_group_kernel, dim3(p.groups), block, 0, s, a);
  launched(hipGetLastError());
}

void beam_reorder(const mit2cfm_kv_cache& c, const mit2cfm_beam_reorder& p, hipStream_t s) {
  check_kv_cache(c);
  need(p.beams >= 1 && p.beams <= (uint32_t)kMaxBeams, "beams must be in [1, 64]");
  need((uint64_t)p.groups * p.beams <= (1u << 20), "groups * beams must be <= 2^20");
  need(p.layers >= 1 && p.layers <= 16384, "layers must be in [1, 16384]");
  need(p.layers == 1 || p.layer_stride % 8 == 0, "layer_stride must be a multiple of 8");
  need(p.parent_stride >= p.beams, "parent_stride must be >= beams");
  if (p.groups == 0) return;
  need(p.parent && p.length && p.table_out, "parent, length and table_out must not be NULL");
  need(p.table_out != c.table, "table_out must not be the cache's table");
  need(p.state == nullptr || (p.state_out && p.state_out != p.state && p.state_words >= 1 && p.state_words < (1u << 31)),
       "state needs a state_out of its own and state_words in [1, 2^31)");
  need(p.token == nullptr || (p.state && p.place), "token needs state and place");
  ReorderArgs a;
  a.k = static_cast<char*>(c.k);
  a.v = static_cast<char*>(c.v);
  a.table = c.table;
  a.table_out = p.table_out;
  a.pages = (int)c.pages;
  a.page_shift = __builtin_ctz(c.page_rows);
  a.kv_heads = (int)c.kv_heads;
  a.table_stride = (int)c.table_stride;
  a.beams = (int)p.beams;
  const int e = kv_elem_bytes(c.dtype);
  a.row16 = (int)c.head_dim * e / 16;
  a.layer16 = p.layers > 1 ? (int64_t)(p.layer_stride * e / 16) : 0;
  a.parent = p.parent;
  a.parent_stride = p.parent_stride;
  a.length = p.length;
  a.state = p.state;
  a.state_out = p.state_out;
  a.state_words = (int)p.state_words;
  a.token = p.token;
  a.place = p.place;
  hipLaunchKernelGGL(reorder_kernel, dim3(p.groups * p.beams, 1 + 2 * p.layers), dim3(kReorderThreads), 0, s, a);
  launched(hipGetLastError());
}

}  // namespace mit2hip
