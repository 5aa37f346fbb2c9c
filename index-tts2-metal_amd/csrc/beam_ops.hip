// beam_ops.hip -- a beam search's step (see beam_ops.h and mit2cfm.h for what
// the operators compute).
#include "beam_ops.h"

#include <algorithm>
#include <cfloat>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "device_common.h"
#include "engine.h"
#include "kv_ops.h"
#include "overlap.h"

namespace mit2hip {

namespace {

typedef __bf16 bf16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
  int beams, vocab, count, stop;
  int splits, chunk;  // of a row's logits: chunk of them, a multiple of 8, a block
  const float* scores;
  const int32_t* finished;
  float* scores_out;
  int32_t *parent_out, *token_out, *finished_out;
  double* sums;    // workspace: [rows][splits] sum of exp(x - max)
  uint64_t* cand;  // [rows][splits][count] the split's best logits, as rank keys
  float* tops;     // [rows][splits] max
};

constexpr int kSelectThreads = 256, kSelectWaves = kSelectThreads / 64;
constexpr int kPerThread = 16;  // logits of a thread
constexpr int kMaxChunk = kSelectThreads * kPerThread;
constexpr int kListed = 2;  // times count: threads of a wave that may list their logits

// A logit as the selection sees it.
template <typename T>
__device__ __forceinline__ float logit(T v) {
  const float x = (float)v;
  return x != x ? -INFINITY : fminf(x, FLT_MAX);
}
// Keys that order as the selection does: larger values first, of equal ones the
// lower index; no key of a logit is 0.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t t) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 counts as 0)
  return (uint64_t)((u & 0x80000000u) ? ~u : u | 0x80000000u) << 32 | (uint32_t)~t;
}
__device__ __forceinline__ float key_logit(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t key_token(uint64_t k) { return ~(uint32_t)k; }

// The order of floats as unsigned integers; of no float 0.
__device__ __forceinline__ uint32_t float_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// The largest number that at least n of a wave's keys, of BITS bits, reach (0: fewer
// than n are over 0), built from its top bit by votes.
template <int BITS>
__device__ __forceinline__ uint32_t reached_by(uint32_t key, int n) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = BITS - 1; bit >= 0; --bit) {
    const uint32_t c = t | 1u << bit;
    t = __popcll(__ballot(key >= c)) >= n ? c : t;
  }
  return t;
}

// The key that a wave's lanes with `has` (some have) share.
__device__ __forceinline__ uint32_t key_of_wave(uint32_t key, bool has) {
  return (uint32_t)__builtin_amdgcn_readlane((int)key, __ffsll((unsigned long long)__ballot(has)) - 1);
}

// Whether a live beam's logits count: it exists and is not finished.
__device__ __forceinline__ bool live(const SelectArgs& a, int r) {
  return a.scores[r] > -INFINITY && !(a.finished && a.finished[r] != 0);
}

// Block (split, row): the split's maximum, the sum of its exponentials and its
// `count` best, of one pass over its logits, which stay in registers.
//
// The best: every thread's largest logit; of each wave's 64 the count-th, by
// votes, and where more than twice that many threads reach it (ties) the lowest
// tokens among them; the largest of those bounds is reached by at least `count`
// logits of the split and by those of few threads a wave, which alone list what
// they have from it on; the few in the list find their ranks by counting.  No order
// of threads or atomics shows in the result.
//
// Bound by its own instructions and waits (votes, barriers, ranks) more than by the
// loads: 14 us for 256 rows of 50001 bf16, whose 26 MB take 6; 5.6 us for three rows of
// 8194, which is one block's way through.  With 32 logits a thread 15 and 6.4 us.
template <typename T>
__global__ __launch_bounds__(kSelectThreads) void select_rows_kernel(SelectArgs a) {
  constexpr int W = 16 / sizeof(T), LOADS = kPerThread / W;  // logits of a load
  struct alignas(16) Load {
    T v[W];
  };
  extern __shared__ uint64_t list[];
  __shared__ uint64_t s_kth[kSelectWaves];
  __shared__ float s_max[kSelectWaves];
  __shared__ double s_sum[kSelectWaves];
  __shared__ uint32_t s_n;
  const int r = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* x = static_cast<const T*>(a.logits) + r * a.row;
  // splits begin on 16 bytes, the first up to W - 1 logits before the row
  const int skew = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  const int begin = split * a.chunk - skew, from = max(begin, 0), to = min(begin + a.chunk, a.vocab);
  float v[kPerThread];  // -inf outside the split
  const int at = begin + tid * W;
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int t0 = at + i * kSelectThreads * W;
    if (t0 >= from && t0 + W <= to) {
      const Load l = *reinterpret_cast<const Load*>(x + t0);
#pragma unroll
      for (int e = 0; e < W; ++e) v[i * W + e] = logit(l.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) v[i * W + e] = t0 + e >= from && t0 + e < to ? logit(x[t0 + e]) : -INFINITY;
    }
  }
  if (!live(a, r)) return;  // its logits do not matter (looked up behind the loads, not before them)
  if (tid == 0) s_n = 0;
  auto token = [&](int k) { return at + k / W * kSelectThreads * W + k % W; };
  auto inside = [&](int k) { return token(k) >= from && token(k) < to; };
  float top = v[0];
#pragma unroll
  for (int k = 1; k < kPerThread; ++k) top = fmaxf(top, v[k]);
  float m = top;
#pragma unroll
  for (int off = 32; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
  // a thread that has any logit: its first load's last, or a later load's first, is inside
  bool any = false;
#pragma unroll
  for (int i = 0; i < LOADS; ++i) any |= at + i * kSelectThreads * W + W > from && at + i * kSelectThreads * W < to;
  // (a 16-bit type's values differ in their upper bits alone; bf16's and FLT_MAX,
  // which stands for +inf, in bit 15 too)
  constexpr int LOW = sizeof(T) == 4 ? 0 : std::is_same<T, half_t>::value ? 13 : 15;
  const uint32_t key = any ? float_key(top) : 0u, high = key >> LOW, t32 = reached_by<32 - LOW>(high, a.count);
  uint64_t kth = (uint64_t)(t32 << LOW) << 32;
  const int over = __popcll(__ballot(high > t32)), ties = __popcll(__ballot(high == t32));
  if (t32 != 0 && over + ties > kListed * a.count) {
    int first = 0;  // the thread's lowest token of that value
#pragma unroll
    for (int k = kPerThread - 1; k >= 0; --k) first = v[k] == top && inside(k) ? token(k) : first;
    constexpr int PLACES = 15;  // of a chunk's tokens, counted from its end
    static_assert(kMaxChunk < 1 << PLACES, "a chunk's tokens fit the search");
    const uint32_t place =
        reached_by<PLACES>(high == t32 ? (uint32_t)(kMaxChunk - (first - begin)) : 0u, a.count - over);
    const uint32_t tied = key_of_wave(key, high == t32);
    kth = (uint64_t)tied << 32 | ~(uint32_t)(begin + kMaxChunk - (int)place);
  }
  if (lane == 0) {
    s_max[wave] = m;
    s_kth[wave] = kth;
  }
  __syncthreads();
  uint64_t least = s_kth[0];
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    least = s_kth[w] > least ? s_kth[w] : least;
    m = fmaxf(m, s_max[w]);
  }
  // (2 to the power of: the argument's rounding is relative to it, and a term that
  // far below the largest weighs as little; a thread's few terms are summed in
  // fp32, in pairs)
  const float base = m == -INFINITY ? 0.f : m;
  float part[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) part[k] = __builtin_amdgcn_exp2f((v[k] - base) * 1.4426950408889634f);
#pragma unroll
  for (int w = kPerThread / 2; w >= 1; w /= 2)
#pragma unroll
    for (int k = 0; k < w; ++k) part[k] += part[k + w];
  double sum = (double)part[0];
#pragma unroll
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, kWave);
  if (lane == 0) s_sum[wave] = sum;
  if (key != 0 && key >= (uint32_t)(least >> 32)) {
    const float bound = (uint32_t)(least >> 32) <= float_key(-INFINITY) ? -INFINITY : key_logit(least);
    uint32_t hits = 0;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) hits |= v[k] >= bound ? 1u << k : 0u;
    const bool one = (hits & (hits - 1)) == 0;  // the thread's largest
    for (; hits; hits &= hits - 1) {
      const int t = token(__ffs(hits) - 1);
      if (t < from || t >= to) continue;
      const uint64_t rk = rank_key(one ? top : logit(x[t]), (uint32_t)t);
      if (rk >= least) list[atomicAdd(&s_n, 1u)] = rk;
    }
  }
  __syncthreads();
  const int n = (int)s_n;
  const size_t out = (size_t)r * a.splits + split;
  for (int j = tid; j < n; j += kSelectThreads) {
    const uint64_t k = list[j];
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += list[o] > k ? 1 : 0;
    if (rank < a.count) a.cand[out * a.count + rank] = k;
  }
  for (int j = n + tid; j < a.count; j += kSelectThreads) a.cand[out * a.count + j] = 0;
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kSelectWaves; ++w) sum += s_sum[w];
    a.sums[out] = sum;
    a.tops[out] = m;
  }
}

// A candidate of a group: its score as a key that orders, and what orders equal
// ones: the lower beam, its larger logit, the lower token (6, 32 and 24 bits).
struct Scored {
  uint64_t s, at;
  __device__ __forceinline__ bool over(const Scored& o) const { return s > o.s || (s == o.s && at < o.at); }
  __device__ __forceinline__ int beam() const { return (int)(at >> 56); }
  __device__ __forceinline__ int token() const { return (int)(at & 0xffffffu); }
};
__device__ __forceinline__ uint64_t score_key(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return (u >> 63) ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double key_score(uint64_t k) {
  return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k));
}
__device__ __forceinline__ Scored scored(double score, int beam, float logit, uint32_t token) {
  return {score_key(score), (uint64_t)beam << 56 | (uint64_t)~float_key(logit) << 24 | token};
}

constexpr int kGroupList = 1024;
constexpr int kGroupThreads = 512, kGroupWaves = kGroupThreads / 64;
constexpr int kHeldCandidates = 4;  // of a thread, kept in registers

// Block (group): the best of its beams' candidates, found as a split's are (by
// the scores rounded to fp32, which keeps their order, until the list is made);
// a list that overflows, as with ties of very many candidates, is worked off one
// by one.  A group's block waits for the chip, not the chip for it: 6.5 us for 32
// groups of 1664 candidates (10 with 256 threads, as much with 1024), 4.4 for 54.
__global__ __launch_bounds__(kGroupThreads) void select_group_kernel(SelectArgs a) {
  __shared__ double s_log[kMaxBeams];   // a beam's logits' log sum; -inf: none is over -inf
  __shared__ float s_cum[kMaxBeams];    // its score
  __shared__ uint8_t s_kind[kMaxBeams]; // bit 0: finished, bit 1: does not exist
  __shared__ Scored list[kGroupList];
  __shared__ Scored s_w[kGroupWaves];
  __shared__ uint32_t s_kth[kGroupWaves];
  __shared__ uint32_t s_n;
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) s_n = 0;
  for (int b = tid >> 4; b < a.beams; b += kGroupThreads / 16) {  // sixteen lanes a beam
    const int r = g * a.beams + b;
    const float cum = a.scores[r];
    const int kind = (cum > -INFINITY ? 0 : 2) | (a.finished && a.finished[r] != 0 ? 1 : 0);
    double log_sum = -INFINITY;
    if (kind == 0) {
      const double* sums = a.sums + (size_t)r * a.splits;
      const float* tops = a.tops + (size_t)r * a.splits;
      float m = -INFINITY;
      for (int s = tid & 15; s < a.splits; s += 16) m = fmaxf(m, tops[s]);
#pragma unroll
      for (int w = 1; w < 16; w *= 2) m = fmaxf(m, __shfl_xor(m, w, kWave));
      double sum = 0.0;
      for (int s = tid & 15; s < a.splits; s += 16)
        if (tops[s] > -INFINITY) sum += sums[s] * exp((double)tops[s] - (double)m);
#pragma unroll
      for (int w = 1; w < 16; w *= 2) sum += __shfl_xor(sum, w, kWave);
      if (m > -INFINITY) log_sum = (double)m + log(sum);
    }
    if ((tid & 15) == 0) {
      s_log[b] = log_sum;
      s_cum[b] = cum;
      s_kind[b] = (uint8_t)kind;
    }
  }
  const int per = a.splits * a.count, n = a.beams * per;
  const Scored none = {0, ~0ull};
  const uint64_t* cand = a.cand + (size_t)g * n;
  // the stored keys of this thread's first candidates, asked for before the sums are known
  uint64_t key[kHeldCandidates];
#pragma unroll
  for (int i = 0; i < kHeldCandidates; ++i) {
    const int c = tid + i * kGroupThreads;
    key[i] = c < n ? cand[c] : 0;  // (what a beam without a pass left there is not used)
  }
  __syncthreads();
  auto candidate = [&](int c, uint64_t stored) -> Scored {
    const int b = c / per, k = c - b * per, kind = s_kind[b];
    if (kind != 0) {  // the lowest tokens at -inf; of a finished beam the stop token before them
      if (k >= a.count || k >= a.vocab) return none;
      const int t = kind & 2 ? k : k == 0 ? a.stop : k - 1 < a.stop ? k - 1 : k;
      return scored(kind == 1 && k == 0 ? (double)s_cum[b] : -INFINITY, b, -INFINITY, (uint32_t)t);
    }
    if (stored == 0) return none;
    // (the logit less the log sum first: beside a huge one, the beam's score would be lost)
    const float x = key_logit(stored);
    return scored(x > -INFINITY ? (double)s_cum[b] + ((double)x - s_log[b]) : -INFINITY, b, x, key_token(stored));
  };
  Scored held[kHeldCandidates];
#pragma unroll
  for (int i = 0; i < kHeldCandidates; ++i) {
    const int c = tid + i * kGroupThreads;
    held[i] = c < n ? candidate(c, key[i]) : none;
  }
  auto each = [&](auto&& f) {  // every candidate of this thread
#pragma unroll
    for (int i = 0; i < kHeldCandidates; ++i) f(held[i]);
    for (int c = tid + kHeldCandidates * kGroupThreads; c < n; c += kGroupThreads) f(candidate(c, cand[c]));
  };
  auto write = [&](const Scored& c, int rank) {
    const size_t at = (size_t)g * a.count + rank;
    const int b = c.beam(), t = c.token();
    a.scores_out[at] = (float)key_score(c.s);
    a.parent_out[at] = b;
    a.token_out[at] = t;
    if (a.finished_out) a.finished_out[at] = t == a.stop || (s_kind[b] & 1) ? 1 : 0;
  };
  auto rounded = [](const Scored& x) { return x.s == 0 ? 0u : float_key((float)key_score(x.s)); };
  uint32_t best = 0;
  each([&](const Scored& x) { best = max(best, rounded(x)); });
  const uint32_t kth = reached_by<32>(best, a.count);
  if (lane == 0) s_kth[wave] = kth;
  __syncthreads();
  uint32_t least = 1;
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) least = max(least, s_kth[w]);
  if (best >= least)
    each([&](const Scored& x) {
      if (rounded(x) < least) return;
      const uint32_t i = atomicAdd(&s_n, 1u);
      if (i < kGroupList) list[i] = x;
    });
  __syncthreads();
  const int m = (int)s_n;
  if (m <= kGroupList) {
    for (int j = tid >> 2; j < m; j += kGroupThreads / 4) {  // four lanes a candidate
      const Scored x = list[j];
      int rank = 0;
#pragma unroll 4
      for (int o = tid & 3; o < m; o += 4) rank += list[o].over(x) ? 1 : 0;
      rank += __shfl_xor(rank, 1, kWave);
      rank += __shfl_xor(rank, 2, kWave);
      if ((tid & 3) == 0 && rank < a.count) write(x, rank);
    }
    return;
  }
  Scored last = {~0ull, 0};
  for (int k = 0; k < a.count; ++k) {
    Scored next = none;
    each([&](const Scored& x) {
      if (last.over(x) && x.over(next)) next = x;
    });
#pragma unroll
    for (int off = 32; off; off >>= 1) {
      const Scored o = {__shfl_xor((unsigned long long)next.s, off, kWave), __shfl_xor((unsigned long long)next.at, off, kWave)};
      if (o.over(next)) next = o;
    }
    __syncthreads();
    if (lane == 0) s_w[wave] = next;
    __syncthreads();
    last = s_w[0];
    for (int w = 1; w < kGroupWaves; ++w)
      if (s_w[w].over(last)) last = s_w[w];
    if (tid == 0) write(last, k);
  }
}

bool select_in_range(const mit2cfm_beam_select& a) {
  return a.dtype >= MIT2CFM_DTYPE_F32 && a.dtype <= MIT2CFM_DTYPE_BF16 && a.beams >= 1 && a.beams <= (uint32_t)kMaxBeams &&
         a.vocab >= 1 && a.vocab <= (1u << 24) && a.count >= 1 && a.count <= (uint32_t)kMaxCount &&
         a.count <= (uint64_t)a.beams * a.vocab && (uint64_t)a.groups * a.beams <= 65535;
}
size_t align16(size_t b) { return (b + 15) & ~size_t(15); }
// A row's logits in even splits of at most kMaxChunk, which begin up to 7 logits
// before it.
int select_splits(uint32_t vocab) { return (int)((vocab + 7 + kMaxChunk - 1) / kMaxChunk); }

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

constexpr int kReorderThreads = 512;

// Block (new beam, part): part 0 writes the beam's table row and states, part 1
// + l copies the part page's rows of layer l, for a beam that is not its
// parent's first child.  Each block finds whose pages are whose by itself, from
// the group's parents as bits: a beam is a further child when an earlier one
// has its parent, its rank among those is its index less the distinct parents
// before it, and there are as many beams without children.
//
// Bound by the part pages' copies: 32 searches of 8 beams, 24 layers of 8 heads of 64
// bf16, 135 MB in 33 us a call (4.1 TB/s; the kernel 27 on pages that the last run
// left in the caches).  Their stores go past the caches, whose lines the
// pages' other bytes would come into first: 45 us with ordinary ones (and no loss to
// the attention after, which reads far more than it finds there).  Three beams of 20
// fp32 heads take 2.9 us, most of it four waits in a row (parents, length, table,
// rows).  Several layers a block, 49 us and more.
constexpr int kCopyBatch = 2;  // 16-byte loads of a thread in flight, of k and of v each
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
  const int64_t layer = (int64_t)(blockIdx.y - 1) * a.layer16, head = (int64_t)a.row16 << a.page_shift;
  const int per = part * a.row16, n = per * a.kv_heads;  // 16-byte vectors: a head's, all
  u32x4 *k = reinterpret_cast<u32x4*>(a.k) + layer, *v = reinterpret_cast<u32x4*>(a.v) + layer;
  const int64_t s = (int64_t)src * a.kv_heads * head, d = (int64_t)dst * a.kv_heads * head;
  for (int i0 = tid; i0 < n; i0 += kReorderThreads * kCopyBatch) {
    u32x4 x[kCopyBatch], y[kCopyBatch];
    int64_t at[kCopyBatch];
#pragma unroll
    for (int u = 0; u < kCopyBatch; ++u) {
      const int i = min(i0 + u * kReorderThreads, n - 1), h = i / per;
      at[u] = h * head + (i - h * per);
      x[u] = k[s + at[u]];
      y[u] = v[s + at[u]];
    }
#pragma unroll
    for (int u = 0; u < kCopyBatch; ++u)
      if (i0 + u * kReorderThreads < n) {
        __builtin_nontemporal_store(x[u], k + d + at[u]);
        __builtin_nontemporal_store(y[u], v + d + at[u]);
      }
  }
}

}  // namespace

uint64_t beam_select_workspace(const mit2cfm_beam_select& a) {
  if (!select_in_range(a)) return 0;
  const size_t parts = (size_t)a.groups * a.beams * select_splits(a.vocab);
  return align16(parts * 8) + align16(parts * a.count * 8) + align16(parts * 4) + 16;
}

void beam_select(const mit2cfm_beam_select& p, hipStream_t s) {
  need(select_in_range(p), "dtype, beams, vocab, count or groups * beams out of range");
  need(p.stop_token >= -1 && (p.stop_token < 0 || (uint32_t)p.stop_token < p.vocab), "stop_token must be -1 or in [0, vocab)");
  need(p.finished == nullptr || p.stop_token >= 0, "finished needs a stop_token");
  if (p.groups == 0) return;
  need(p.logits && p.scores && p.scores_out && p.parent_out && p.token_out,
       "logits, scores, scores_out, parent_out and token_out must not be NULL");
  need(aligned(p.logits, (size_t)kv_elem_bytes(p.dtype)), "logits must be aligned to its type");
  const uint64_t in_bytes = (uint64_t)p.groups * p.beams * 4, out_bytes = (uint64_t)p.groups * p.count * 4;
  need(!meet(p.scores, in_bytes, p.scores_out, out_bytes) &&
           !(p.finished && p.finished_out && meet(p.finished, in_bytes, p.finished_out, out_bytes)),
       "scores_out must not overlap scores, nor finished_out finished");
  need(aligned(p.scores, 4) && aligned(p.finished, 4) && aligned(p.scores_out, 4) && aligned(p.parent_out, 4) &&
           aligned(p.token_out, 4) && aligned(p.finished_out, 4),
       "scores, finished and the outputs must be 4-byte aligned");
  need(p.workspace && p.workspace_bytes >= beam_select_workspace(p), "workspace is NULL or too small");
  need(aligned(p.workspace, 16), "workspace must be 16-byte aligned");
  SelectArgs a;
  a.logits = p.logits;
  a.row = (int64_t)p.logits_row;
  a.beams = (int)p.beams; a.vocab = (int)p.vocab; a.count = (int)p.count;
  a.stop = p.stop_token;
  a.splits = select_splits(p.vocab);
  a.chunk = (int)((p.vocab + 7 + a.splits - 1) / a.splits + 7) / 8 * 8;
  a.scores = p.scores; a.finished = p.finished;
  a.scores_out = p.scores_out; a.parent_out = p.parent_out; a.token_out = p.token_out; a.finished_out = p.finished_out;
  const uint32_t rows = p.groups * p.beams;
  const size_t parts = (size_t)rows * a.splits;
  char* w = static_cast<char*>(p.workspace);
  a.sums = reinterpret_cast<double*>(w);
  w += align16(parts * 8);
  a.cand = reinterpret_cast<uint64_t*>(w);
  w += align16(parts * a.count * 8);
  a.tops = reinterpret_cast<float*>(w);
  const dim3 grid(a.splits, rows), block(kSelectThreads);
  // the list holds all logits of as many threads a wave as may list them
  const size_t lds = std::min<size_t>((size_t)kSelectWaves * kListed * a.count * kPerThread, kMaxChunk) * 8;
  if (p.dtype == MIT2CFM_DTYPE_F32)
    hipLaunchKernelGGL((select_rows_kernel<float>), grid, block, lds, s, a);
  else if (p.dtype == MIT2CFM_DTYPE_F16)
    hipLaunchKernelGGL((select_rows_kernel<half_t>), grid, block, lds, s, a);
  else
    hipLaunchKernelGGL((select_rows_kernel<bf16_t>), grid, block, lds, s, a);
  launched(hipGetLastError());
  hipLaunchKernelGGL(select_group_kernel, dim3(p.groups), dim3(kGroupThreads), 0, s, a);
  launched(hipGetLastError());
}

void beam_reorder(const mit2cfm_kv_cache& c, const mit2cfm_beam_reorder& p, hipStream_t s) {
  check_kv_cache(c);
  need(p.beams >= 1 && p.beams <= (uint32_t)kMaxBeams, "beams must be in [1, 64]");
  need((uint64_t)p.groups * p.beams <= (1u << 20), "groups * beams must be <= 2^20");
  need(p.layers >= 1 && p.layers <= 16384, "layers must be in [1, 16384]");
  need(p.layers == 1 || p.layer_stride % 8 == 0, "layer_stride must be a multiple of 8");
  need(p.layers == 1 || p.layer_stride >= (uint64_t)c.pages * c.kv_heads * c.page_rows * c.head_dim,
       "layer_stride is smaller than a layer");
  need(p.parent_stride >= p.beams, "parent_stride must be >= beams");
  if (p.groups == 0) return;
  need(p.parent && p.length && p.table_out, "parent, length and table_out must not be NULL");
  const uint64_t table_bytes = (uint64_t)p.groups * p.beams * c.table_stride * 4;
  need(!meet(c.table, table_bytes, p.table_out, table_bytes), "table_out overlaps the cache's table");
  need(p.state == nullptr || (p.state_out && p.state_words >= 1 && p.state_words < (1u << 31)),
       "state needs a state_out and state_words in [1, 2^31)");
  const uint64_t state_bytes = (uint64_t)p.groups * p.beams * p.state_words * 4;
  need(p.state == nullptr || !meet(p.state, state_bytes, p.state_out, state_bytes), "state_out overlaps state");
  need(p.token == nullptr || (p.state && p.place), "token needs state and place");
  need(aligned(p.parent, 4) && aligned(p.length, 4) && aligned(p.table_out, 4) && aligned(p.state, 4) &&
           aligned(p.state_out, 4) && aligned(p.token, 4) && aligned(p.place, 4),
       "parent, length, table_out, the states, token and place must be 4-byte aligned");
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
  hipLaunchKernelGGL(reorder_kernel, dim3(p.groups * p.beams, 1 + p.layers), dim3(kReorderThreads), 0, s, a);
  launched(hipGetLastError());
}

}  // namespace mit2hip
