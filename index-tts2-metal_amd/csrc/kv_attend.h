// kv_attend.h -- attention of new rows over a paged cache (kv_ops.h): the kernels
// of one element type, instantiated in kv_attend_{f32,f16,bf16}.hip.
//
// Everything below works on tiles of 16 query rows, a sequence's new rows x the
// query heads of one key head in that order, and of KT keys.  The products are
// transposed: S^T = K Q^T leaves a lane with one query (lane % 16) and, of each 16
// keys, those from 4 (lane / 16) on, which are the slots its group feeds to
// O^T += V^T P: the probabilities never cross lanes.  A lane reads D/16
// neighbouring elements of each of its keys' values and turns them into operands
// by itself, output row i of product d being element (D/16) i + d; at the end
// it holds D/4 neighbouring elements of its query's output.
#pragma once

#include "device_common.h"
#include <climits>
#include <type_traits>

#include "kv_plan.h"
#include "kv_view.h"

namespace mit2hip {

struct AttendArgs {
  CacheView c;
  RowView r;
  const char* q;
  char* out;
  int64_t q_row, q_head, o_row, o_head;
  const uint32_t* mask;
  int mask_words, q_heads, group;
  int q_wide, o_wide;  // rows of q (of out) may be read (written) 16 bytes at a time
  int flip;            // the scale is negative: queries change sign
  float scale2;        // |scale| log2(e): scores in powers of two
};

// Attention of sequences that share their first rows (kv_prefix.h), in one launch: first
// the blocks of the shared rows, each for new rows of all a group's sequences, then
// those of what each sequence has of its own.  Both leave parts, for one join.
struct PrefixArgs : AttendArgs {
  const int32_t* bounds;  // [groups + 1] first sequences of the groups
  const int32_t* shared;  // [groups] rows that a group's sequences share
  int groups;
  int step;               // shared rows are taken in whole runs of this
  AttendPlan own;         // (the kernels' plan is the shared rows')
  uint32_t shared_blocks, blocks;
  size_t pairs;           // query rows x heads
};

template <typename A>
constexpr bool is_prefix = std::is_same<A, PrefixArgs>::value;
template <typename A>
constexpr int wide_blocks = is_prefix<A> ? 3 : 2;  // of a CU

// What splits leave for their join: [row][query head][split] outputs, maxima and
// weights' sums, [row][query head] the number of splits.
struct Parts {
  float* o;
  float2* ml;
  int32_t* n;
};

// Launches a plan's kernels; throws HipError.
void launch_attend_f32(const AttendArgs& a, const AttendPlan& plan, int D, void* workspace, hipStream_t s);
void launch_attend_f16(const AttendArgs& a, const AttendPlan& plan, int D, void* workspace, hipStream_t s);
void launch_attend_bf16(const AttendArgs& a, const AttendPlan& plan, int D, void* workspace, hipStream_t s);

#if defined(KV_ATTEND_KERNELS)

// The matrix instruction of a type: its operand, and the keys of a tile.
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

// The sizes that follow from a type and a head size.
template <typename T, int D_>
struct Dims {
  static constexpr int D = D_, DP = D / 16;
  static constexpr int KT = Mat<T>::KT, NT = KT / 16;
  static constexpr int DC = sizeof(T) == 2 ? D / 32 : D / 4;  // steps of a score's product
  static constexpr int NV = KT / 4;                           // a lane's keys of a tile
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A lane's key number e of a tile (grp = lane / 16).
__device__ __forceinline__ int key_of(int e, int grp) { return 16 * (e >> 2) + 4 * grp + (e & 3); }

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

// Keys of a split of a sequence of len keys.
__device__ __forceinline__ int chunk_of(int len, int chunk, int splits) {
  const int least = (max(len, 0) + splits - 1) / splits, step = chunk_step(false);
  return max(chunk, (least + step - 1) / step * step);
}

// The sequence that tile number t of the whole batch (of `mtile` query rows)
// belongs to, its number there, the sequence's bounds and its length; false past
// the last.  A wave's lanes look at 64 sequences at a time.
struct Found {
  int seq, in_seq, start, stop, length;
};
__device__ __forceinline__ bool find_tile(const RowView& r, int group, int mtile, int t, Found& f) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < r.seqs; base += 64) {
    int n = 0, s0 = 0, s1 = 0, length = 0;
    if (base + lane < r.seqs) {
      s0 = r.start[base + lane];
      s1 = r.start[base + lane + 1];
      length = r.length[base + lane];
      const int rows = min(s1, r.rows) - max(s0, 0);
      n = rows > 0 ? (int)(((int64_t)rows * group + mtile - 1) / mtile) : 0;
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
      f.seq = __builtin_amdgcn_readfirstlane(base + l);
      f.in_seq = t - before - __builtin_amdgcn_readlane(incl - n, l);
      f.start = __builtin_amdgcn_readlane(s0, l);
      f.stop = __builtin_amdgcn_readlane(s1, l);
      f.length = __builtin_amdgcn_readlane(length, l);
      return true;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// A block's part of the work: a tile of query rows, a key head, a split of the keys.
// Workgroups go to the 8 XCDs in turn.  by_xcd: units of a key head and split are
// dealt to the XCDs and their tiles follow each other there, so that those of
// one sequence find its keys in that XCD's L2.
struct Part {
  int seq, kvh, split;
  int start, raw_start;  // the sequence's first new row in the buffers, and as given
  int mrows, m0;         // the sequence's query rows; the tile's first
  int first, len;        // cached rows before the new ones, and all
  int begin, end;        // the split's keys
  int parts;             // splits that hold keys
  bool whole;            // one split holds all keys: results are final
  bool own;              // (of shared prefixes) a sequence's own rows
};
__device__ __forceinline__ bool find_part(const AttendArgs& a, const AttendPlan& plan, int mtile, Part& p) {
  int tile = blockIdx.x, unit = blockIdx.y;
  if (plan.by_xcd) {
    const int slot = blockIdx.x >> 3;
    unit = slot / plan.tiles * 8 + (blockIdx.x & 7);
    tile = slot % plan.tiles;
    if (unit >= a.c.kv_heads * plan.splits) return false;
  }
  p.kvh = unit % a.c.kv_heads;
  p.split = unit / a.c.kv_heads;
  Found f;
  if (!find_tile(a.r, a.group, mtile, tile, f)) return false;
  p.seq = f.seq;
  p.raw_start = f.start;
  const int stop = f.stop, length = f.length;
  p.start = max(p.raw_start, 0);
  p.mrows = (min(stop, a.r.rows) - p.start) * a.group;
  p.m0 = f.in_seq * mtile;
  p.first = length - (stop - p.raw_start);
  p.len = min(length, a.c.capacity());
  const int chunk = chunk_of(p.len, plan.chunk, plan.splits);
  p.begin = p.split * chunk;
  p.end = min(p.begin + chunk, p.len);
  p.whole = p.len <= chunk;
  p.parts = p.whole ? 1 : (p.len + chunk - 1) / chunk;
  return p.split == 0 || p.begin < p.len;
}

// Where a split's part goes, and how many of them there are.
__device__ __forceinline__ size_t slot_of(const AttendArgs&, const AttendPlan& plan, const Part& p, size_t pair) {
  return pair * plan.splits + p.split;
}
__device__ __forceinline__ void tell_parts(const AttendArgs&, const AttendPlan& plan, const Part& p, const Parts& part, size_t pair) {
  if (p.split == 0 && plan.splits > 1) part.n[pair] = p.parts;
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int off = 32; off; off >>= 1) x = min(x, __shfl_xor(x, off, kWave));
  return __builtin_amdgcn_readfirstlane(x);
}
// Of 64 (or fewer) runs of n tiles, lane by lane: the one that holds tile t, and the
// tiles before it; -1: none does, `before` then counts them all.
__device__ __forceinline__ int run_of(int n, int t, int& before) {
  const int lane = threadIdx.x & 63;
  int incl = n;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(incl, off, kWave);
    if (lane >= off) incl += o;
  }
  const uint64_t past = __ballot(before + incl > t);
  if (!past) {
    before += __builtin_amdgcn_readlane(incl, 63);
    return -1;
  }
  const int l = __ffsll((unsigned long long)past) - 1;
  before += __builtin_amdgcn_readlane(incl - n, l);
  return l;
}
__device__ __forceinline__ int tiles_of(const AttendArgs& a, int start, int stop, int mtile) {
  const int rows = min(stop, a.r.rows) - max(start, 0);
  return rows > 0 ? (int)(((int64_t)rows * a.group + mtile - 1) / mtile) : 0;
}

// What a wave's lanes hold of the sequences and groups where neither are more than 64:
// asked for at once (looked up one from the other, they are three waits in a row).
struct Few {
  bool all;                 // they are no more
  int start, stop, length;  // sequence `lane`'s
  int lo, hi, said;         // group `lane`'s
  __device__ __forceinline__ Few(const PrefixArgs& a) {
    const int lane = threadIdx.x & 63;
    all = a.r.seqs <= 64 && a.groups <= 64;
    start = stop = length = lo = hi = said = 0;
    if (!all) return;
    const int s = min(lane, a.r.seqs - 1);
    start = a.r.start[s];
    stop = a.r.start[s + 1];
    length = a.r.length[s];
    if (a.groups > 0) {
      const int g = min(lane, a.groups - 1);
      lo = a.bounds[g];
      hi = a.bounds[g + 1];
      said = a.shared[g];
    }
    if (lane >= a.r.seqs) start = stop = 0;
    if (lane >= a.groups) lo = hi = 0;
  }
};

// Rows that the sequences lo .. hi - 1 may share: as many as said, of those before any
// of their new rows, in whole runs of `step`; and the first of them that has new rows (-1:
// none), whose pages are read: the others' may be anything.  (The same for all lanes.)
struct Sharing {
  int rows, reader;
};
__device__ __forceinline__ Sharing shared_rows(const PrefixArgs& a, const Few& few, int lo, int hi, int said) {
  const int lane = threadIdx.x & 63;
  int least = min(said, a.c.capacity()), reader = -1;
  auto look = [&](int base, bool in, int start, int stop, auto&& length) {
    in = in && stop > start;
    if (in) least = min(least, length() - (stop - start));
    const uint64_t have = __ballot(in);
    if (have && reader < 0) reader = base + __ffsll((unsigned long long)have) - 1;
  };
  if (few.all) {
    look(0, lane >= lo && lane < hi, few.start, few.stop, [&] { return few.length; });
  } else {
    for (int base = lo; base < hi; base += 64) {
      const int s = min(base + lane, hi - 1);
      look(base, base + lane < hi, a.r.start[s], a.r.start[s + 1], [&] { return a.r.length[s]; });
    }
  }
  return {max(wave_min(least), 0) & -a.step, reader};
}
// A sequence's own rows (see Part).
__device__ __forceinline__ bool find_own(const PrefixArgs& a, const Few& few, int mtile, int tile, Part& p) {
  const int lane = threadIdx.x & 63;
  Found f;
  if (few.all) {
    int before = 0;
    const int l = run_of(tiles_of(a, few.start, few.stop, mtile), tile, before);
    if (l < 0) return false;
    f.seq = l;
    f.in_seq = tile - before;
    f.start = __builtin_amdgcn_readlane(few.start, l);
    f.stop = __builtin_amdgcn_readlane(few.stop, l);
    f.length = __builtin_amdgcn_readlane(few.length, l);
  } else if (!find_tile(a.r, a.group, mtile, tile, f)) {
    return false;
  }
  p.seq = f.seq;
  p.raw_start = f.start;
  p.start = max(f.start, 0);
  p.mrows = (min(f.stop, a.r.rows) - p.start) * a.group;
  p.m0 = f.in_seq * mtile;
  p.first = f.length - (f.stop - f.start);
  p.len = min(f.length, a.c.capacity());
  int from = 0;  // the group's shared rows
  for (int base = 0; base < a.groups; base += 64) {
    int lo = few.lo, hi = few.hi, said = few.said;
    if (!few.all) {
      lo = hi = 0;
      if (base + lane < a.groups) {
        lo = a.bounds[base + lane];
        hi = a.bounds[base + lane + 1];
        said = a.shared[base + lane];
      }
    }
    const uint64_t mine = __ballot(lo <= f.seq && f.seq < hi);
    if (!mine) continue;
    const int l = __ffsll((unsigned long long)mine) - 1;
    from = shared_rows(a, few, max(__builtin_amdgcn_readlane(lo, l), 0), min(__builtin_amdgcn_readlane(hi, l), a.r.seqs),
                       __builtin_amdgcn_readlane(said, l)).rows;
    break;
  }
  const int chunk = chunk_of(p.len - from, a.own.chunk, a.own.splits);
  p.begin = min(from + p.split * chunk, max(p.len, from));
  p.end = min(p.begin + chunk, p.len);
  // (bit 16: there are shared rows)
  p.parts = max(1, (p.len - from + chunk - 1) / chunk) | (from > 0 ? 1 << 16 : 0);
  return p.split == 0 || p.begin < p.len;
}
// A group's shared rows: its new rows are as one sequence's, and see all of them.
__device__ __forceinline__ bool find_shared(const PrefixArgs& a, const AttendPlan& plan, const Few& few, int mtile, int tile, Part& p) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < a.groups; base += 64) {
    int lo = few.lo, hi = few.hi, said = few.said, start = 0, stop = 0;
    if (!few.all) {
      lo = hi = 0;
      if (base + lane < a.groups) {
        lo = a.bounds[base + lane];
        hi = a.bounds[base + lane + 1];
        said = a.shared[base + lane];
      }
    }
    lo = max(lo, 0);
    hi = min(hi, a.r.seqs);
    const bool some = lo < hi && said >= a.step;
    if (few.all) {
      start = __shfl(few.start, lo & 63, kWave);
      stop = __shfl(few.stop, (hi - 1) & 63, kWave);
    } else if (some) {
      start = a.r.start[lo];
      stop = a.r.start[hi];
    }
    const int l = run_of(some ? tiles_of(a, start, stop, mtile) : 0, tile, before);
    if (l < 0) continue;
    p.raw_start = __builtin_amdgcn_readlane(start, l);
    p.start = max(p.raw_start, 0);
    p.mrows = (min(__builtin_amdgcn_readlane(stop, l), a.r.rows) - p.start) * a.group;
    p.m0 = (tile - before) * mtile;
    const Sharing of = shared_rows(a, few, __builtin_amdgcn_readlane(lo, l), __builtin_amdgcn_readlane(hi, l), __builtin_amdgcn_readlane(said, l));
    p.seq = max(of.reader, 0);
    p.len = p.first = of.rows;
    const int chunk = chunk_of(p.len, plan.chunk, plan.splits);
    p.begin = p.split * chunk;
    p.end = min(p.begin + chunk, p.len);
    p.parts = (p.len + chunk - 1) / chunk;
    return p.begin < p.len;
  }
  return false;
}
__device__ __forceinline__ bool find_part(const PrefixArgs& a, const AttendPlan& shared, int mtile, Part& p) {
  uint32_t id = blockIdx.y * gridDim.x + blockIdx.x;
  if (id >= a.blocks) return false;
  const Few few(a);
  p.own = id >= a.shared_blocks;
  if (p.own) id -= a.shared_blocks;
  const AttendPlan& plan = p.own ? a.own : shared;
  int tile = id % plan.tiles, unit = id / plan.tiles;
  if (plan.by_xcd) {
    const int slot = id >> 3;
    unit = slot / plan.tiles * 8 + (id & 7);
    tile = slot % plan.tiles;
    if (unit >= a.c.kv_heads * plan.splits) return false;
  }
  p.kvh = unit % a.c.kv_heads;
  p.split = unit / a.c.kv_heads;
  p.whole = false;
  return p.own ? find_own(a, few, mtile, tile, p) : find_shared(a, shared, few, mtile, tile, p);
}
__device__ __forceinline__ size_t slot_of(const PrefixArgs& a, const AttendPlan& shared, const Part& p, size_t pair) {
  return pair * (shared.splits + a.own.splits) + (p.own ? shared.splits : 0) + p.split;
}
__device__ __forceinline__ void tell_parts(const PrefixArgs& a, const AttendPlan&, const Part& p, const Parts& part, size_t pair) {
  if (p.split == 0) part.n[pair + (p.own ? a.pairs : 0)] = p.parts;
}

// A lane's query: its row in the buffers, its place among the sequence's new
// rows (as given), its head.
struct Query {
  int row, i, h;
  __device__ __forceinline__ Query(const AttendArgs& a, const Part& p, int m) {
    const int n = m / a.group;
    row = p.start + n;
    i = row - p.raw_start;
    h = p.kvh * a.group + (m - n * a.group);
  }
};

// The operands of a lane's query.
template <typename T, int D>
__device__ __forceinline__ void load_query(const AttendArgs& a, const Query& x, int grp, typename Mat<T>::op (&qv)[Dims<T, D>::DC]) {
  typedef typename Mat<T>::op Op;
  const T* q = reinterpret_cast<const T*>(a.q) + x.row * a.q_row + x.h * a.q_head;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int c = 0; c < Dims<T, D>::DC; ++c) {
      if (a.q_wide) {
        qv[c] = *reinterpret_cast<const Op*>(q + 32 * c + 8 * grp);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qv[c][e] = q[32 * c + 8 * grp + e];
      }
      if (a.flip) qv[c] = -qv[c];
    }
  } else {
#pragma unroll
    for (int c = 0; c < Dims<T, D>::DC; ++c) qv[c] = a.flip ? -q[D / 4 * grp + c] : q[D / 4 * grp + c];
  }
}

// Which of a lane's keys of the tile at j0 its query sees, of those there (bits).
// Selects only: a branch here (the mask's bit looked up only where it counts)
// was compiled to leave all scores as they were.
template <int NV>
__device__ __forceinline__ uint32_t seen_keys(const AttendArgs& a, const Query& x, int j0, int first, int grp,
                                              uint32_t there) {
  const uint32_t* words = a.mask + (size_t)x.row * a.mask_words;
  uint32_t open = 0;
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    const int n = j0 + key_of(e, grp) - first;
    uint32_t ok = n <= x.i ? 1u : 0u;
    if (a.mask) {
      const int w = n >> 5;
      ok = words[min(max(w, 0), a.mask_words - 1)] >> (n & 31) & 1u;
      ok = n < 0 ? 1u : w < a.mask_words ? ok : 0u;
    }
    open |= ok << e;
  }
  return there & open;
}
// The same for one key.
__device__ __forceinline__ bool sees(const AttendArgs& a, const Query& x, int j, int first) {
  const int n = j - first, w = n >> 5;
  if (n < 0) return true;
  if (!a.mask) return n <= x.i;
  return w < a.mask_words && (a.mask[(size_t)x.row * a.mask_words + w] >> (n & 31) & 1u);
}

// What a wave keeps of 16 queries while it goes over the keys: the running
// maximum (of the scores in powers of two), this lane's share of the weights'
// sum, and the outputs.
//
// The maximum is raised only when a score passes it by kSlack (a wave-wide
// vote): up to there the probabilities, at most 2^kSlack, stay exact in fp32 sums
// and in range as 16-bit operands (add_values); the sum of the weights keeps fp32.
//
// f16's weights are 2^7 times theirs throughout, the sum's too: with the slack up to
// 2^15, in range, and normal down to 2^-21 of the largest.  (As they were, many
// keys that are light beside one, e^-18 of it, added up to nothing.)
constexpr float kSlack = 8.f;
template <typename T>
constexpr float kLift = std::is_same<T, half_t>::value ? 7.f : 0.f;

template <typename T, int D>
struct Running {
  typedef Dims<T, D> S;
  float mx, l;
  floatx4 o[S::DP];
  __device__ __forceinline__ void clear() {
    mx = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < S::DP; ++d) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  // Scores to weights; the outputs so far follow a raised maximum.
  __device__ __forceinline__ void weigh(float (&s)[S::NV], float c2) {
    float top = s[0];
#pragma unroll
    for (int e = 1; e < S::NV; ++e) top = fmaxf(top, s[e]);
    top *= c2;
    if (__any(top > mx + kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float mn = fmaxf(mx, top);
      const float alpha = mn == -INFINITY ? 1.f : exp2f(mx - mn);
      mx = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < S::DP; ++d) o[d] *= alpha;
    }
    const float base = mx == -INFINITY ? 0.f : kLift<T> - mx;
#pragma unroll
    for (int e = 0; e < S::NV; ++e) {
      s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c2, base));
      l += s[e];
    }
  }
  __device__ __forceinline__ float sum() const {
    float x = l + __shfl_xor(l, 16, kWave);
    return x + __shfl_xor(x, 32, kWave);
  }
};

// A tile's scores of 16 queries; `some`: not all keys are seen.
template <typename T, int D>
__device__ __forceinline__ void score_tile(const typename Mat<T>::op (&kv)[Dims<T, D>::NT][Dims<T, D>::DC],
                                           const typename Mat<T>::op (&qv)[Dims<T, D>::DC], bool some, uint32_t seen,
                                           float (&s)[Dims<T, D>::NV]) {
  typedef Dims<T, D> S;
#pragma unroll
  for (int t = 0; t < S::NT; ++t) {
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < S::DC; ++c) acc = Mat<T>::mul(kv[t][c], qv[c], acc);
#pragma unroll
    for (int r = 0; r < 4; ++r) s[4 * t + r] = acc[r];
  }
  if (some) {
#pragma unroll
    for (int e = 0; e < S::NV; ++e) s[e] = seen >> e & 1u ? s[e] : -INFINITY;
  }
}
// A tile's values, weighted, into the outputs of MT x 16 queries.  16-bit operands
// hold a weight rounded to the type; WHOLE: what that leaves off is a second product
// (again rounded: 2^-16 of the weight in bf16, 2^-22 in f16), and errors against 64
// bits are the result's rounding.  One query tile a wave waits for memory, and takes
// it: 64 tokens over up to 8191 bf16 keys 297 us with it, 294 without, one over 131001
// 103 and 102.  Two tiles do not (24 rows of 20 f16 heads of 64 over 3000 keys 39 us,
// not 36), nor does the block form (trees of 63 rows over up to 4099 f16 keys 68, not
// 59; a bf16 prompt of 2047 90, not 75).  Shared prefixes have it in all forms, so that a token's
// precision does not hang on its group's size: 64 tokens on 8191 shared bf16 rows 48 us, not
// 44, trees of up to 9 rows 60, not 55, prompts of 300 rows 395, not 346.
//
// INF: an infinite value's product stays as the first left it: what is left of its weight, 0
// or less, is no part of it.  Without, the outputs' last step sees to it (infinities).
template <typename T, int D, int MT, bool WHOLE, bool INF = true>
__device__ __forceinline__ void add_values(const Piece<T, Dims<T, D>::DP> (&vv)[Dims<T, D>::NV],
                                           const float (&s)[MT][Dims<T, D>::NV], Running<T, D>* run) {
  typedef Dims<T, D> S;
  if constexpr (sizeof(T) == 2) {
    typename Mat<T>::op p[MT], left[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[mt][e] = (T)s[mt][e];
        if (WHOLE) left[mt][e] = (T)(s[mt][e] - (float)p[mt][e]);
      }
#pragma unroll
    for (int d = 0; d < S::DP; ++d) {
      typename Mat<T>::op v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = vv[e].v[d];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        run[mt].o[d] = Mat<T>::mul(v, p[mt], run[mt].o[d]);
        if (WHOLE) {
          const floatx4 more = Mat<T>::mul(v, left[mt], run[mt].o[d]);
#pragma unroll
          for (int r = 0; r < 4; ++r) run[mt].o[d][r] = !INF || finite(more[r]) ? more[r] : run[mt].o[d][r];
        }
      }
    }
  } else {
#pragma unroll
    for (int d = 0; d < S::DP; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) run[mt].o[d] = Mat<T>::mul(vv[e].v[d], s[mt][e], run[mt].o[d]);
  }
}

// New rows' values that are not finite must not meet a weight of 0 (0 x NaN
// would reach rows that do not see them): they enter the products as 0 and join
// at the end, for the rows that see them.  Rows before the new ones, which every
// row sees, stay in the products (new0: the tile's first key's place among the
// new rows, negative before them).
template <typename T, int NV, int DP>
__device__ __forceinline__ bool take_out(Piece<T, DP> (&vv)[NV], int new0, int grp) {
  bool odd = false;
#pragma unroll
  for (int e = 0; e < NV; ++e)
#pragma unroll
    for (int d = 0; d < DP; ++d) {
      const bool bad = new0 + key_of(e, grp) >= 0 && !finite(vv[e].v[d]);
      vv[e].v[d] = bad ? (T)0.f : vv[e].v[d];
      odd = odd | bad;
    }
  return __any(odd);
}
// Calls f(v) with the values of each of the split's new rows that query x sees.
template <typename T, int D, typename F>
__device__ __forceinline__ void put_back(const AttendArgs& a, const Part& p, const Query& x, F&& f) {
  for (int j = max(p.begin, max(p.first, 0)); j < p.end; ++j) {
    const int page = a.c.page_of(p.seq, j);
    if (page < 0 || !sees(a, x, j, p.first)) continue;
    f(reinterpret_cast<const T*>(a.c.v) + a.c.row_in(page, j, D) + p.kvh * a.c.head_stride(D));
  }
}
// What a value that was taken out adds.
template <typename T>
__device__ __forceinline__ float taken_out(T v) {
  return finite(v) ? 0.f : (float)v;
}
// Outputs that infinite values made NaN: what is left of a weight, 0 or less, times them.
// Where an output is not finite, the values that stayed in the products, of the split's rows
// before `end` (all of them seen by all of the wave's queries), are looked at again, every
// 16th row by a lane: with one infinite value 64 tokens on 8191 shared bf16 rows take 142 us,
// without 50.
template <typename T, int D>
__device__ __forceinline__ void infinities(const AttendArgs& a, const Part& p, int end, floatx4 (&o)[Dims<T, D>::DP], float weights) {
  constexpr int DP = Dims<T, D>::DP;
  const int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), lq = lane & 15, grp = lane >> 4;  // (not held until here)
  bool odd = false;
#pragma unroll
  for (int d = 0; d < DP; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) odd = odd | !finite(o[d][r]);
  odd = odd && finite(weights);
  if (!__any(odd)) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {  // (one after the other, for fewer registers)
    float met[DP];
#pragma unroll
    for (int d = 0; d < DP; ++d) met[d] = 0.f;
    for (int j = p.begin + lq; j < end; j += 16) {
      const int page = a.c.page_of(p.seq, j);
      if (page < 0) continue;
      const T* v = reinterpret_cast<const T*>(a.c.v) + a.c.row_in(page, j, D) + p.kvh * a.c.head_stride(D) + D / 4 * grp + DP * r;
      const Piece<T, DP> x = *reinterpret_cast<const Piece<T, DP>*>(v);
#pragma unroll
      for (int d = 0; d < DP; ++d) met[d] += taken_out(x.v[d]);
    }
#pragma unroll
    for (int d = 0; d < DP; ++d) {
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) met[d] += __shfl_xor(met[d], off, kWave);
      o[d][r] = odd && met[d] != 0.f ? met[d] : o[d][r];
    }
  }
}

// Few query rows: 16 MT of them a block, whose waves take every fourth tile of
// the split's keys and join at the end.  Bound by the keys and values, which go
// from memory straight into operands: nothing passes LDS until the join.
// BIG: a tile of keys lies in one page, whose entry is the same for all lanes.
//
// 64 tokens over up to 8191 bf16 keys of 8 heads of 128, in pages of 16: 1.52 GB in 288 us
// (5.3 TB/s; a large copy reaches 4.7); one over 131001, 537 MB in 96 us (5.6).  Three
// tokens over 703 fp32 keys of 20 heads of 64 take 8.2 us, 5.6 of them the way to the
// first key and from the last: sequence, page, keys, the join in LDS.
template <typename T, int D, int MT, bool BIG, typename A>
__global__ __launch_bounds__(kAttendThreads) void attend_kernel(A a, AttendPlan plan, Parts part) {
  typedef Dims<T, D> S;
  typedef typename Mat<T>::op Op;
  constexpr int KT = S::KT, NT = S::NT, DP = S::DP, DC = S::DC, NV = S::NV;
  __shared__ float sO[kAttendWaves][16][D + 4];
  __shared__ float2 sML[kAttendWaves][16];
  __shared__ int s_dirty;

  Part p;
  if (!find_part(a, plan, 16 * MT, p)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 15, grp = lane >> 4;
  if (tid == 0) s_dirty = 0;
  __syncthreads();

  const int64_t head = p.kvh * a.c.head_stride(D);
  const T* K = reinterpret_cast<const T*>(a.c.k) + head;
  const T* V = reinterpret_cast<const T*>(a.c.v) + head;
  const int32_t* table = a.c.table + (size_t)p.seq * a.c.table_stride;
  const int pmask = (1 << a.c.page_shift) - 1;
  const int64_t page_elems = ((int64_t)a.c.kv_heads << a.c.page_shift) * D;
  // not BIG: lane i (of the first KT) has key i's entry
  auto entry = [&](int j0) {
    const int j = BIG ? j0 : j0 + (lane & (KT - 1));
    const int e = table[min(j, p.len - 1) >> a.c.page_shift];
    return (unsigned)e < (unsigned)a.c.pages && j < p.len ? e : -1;
  };
  int next = p.begin + KT * wave < p.end ? entry(p.begin + KT * wave) : -1;

  int qm[MT];
  Op qv[MT][DC];
  Running<T, D> run[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    qm[mt] = min(p.m0 + 16 * mt + lq, p.mrows - 1);
    load_query<T, D>(a, Query(a, p, qm[mt]), grp, qv[mt]);
    run[mt].clear();
  }
  bool dirty = false;

  for (int j0 = p.begin + KT * wave; j0 < p.end; j0 += KT * kAttendWaves) {
    const int page = next;
    if (j0 + KT * kAttendWaves < p.end) next = entry(j0 + KT * kAttendWaves);
    if (BIG ? page < 0 : !__any(page >= 0)) continue;
    // operands (rows past the end read the last one's place; they count as unseen)
    Op kv[NT][DC];
    Piece<T, DP> vv[NV];
    uint32_t there;  // bit e: this lane's key e is
    const T *kp[NT], *vp[NV];
    if (BIG) {
      const T* kt = K + page * page_elems;
      const T* vt = V + page * page_elems;
      const int r0 = j0 & pmask, last = min(KT, p.len - j0) - 1;
#pragma unroll
      for (int t = 0; t < NT; ++t) kp[t] = kt + (r0 + min(16 * t + lq, last)) * D;
      there = 0;
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        vp[e] = vt + (r0 + min(key_of(e, grp), last)) * D;
        there |= (key_of(e, grp) <= last ? 1u : 0u) << e;
      }
    } else {
      there = 0;
      auto at = [&](int key, const T* base, bool& ok) {
        const int e = __shfl(page, key, kWave);
        ok = e >= 0;
        return base + max(e, 0) * page_elems + ((j0 + key) & pmask) * D;
      };
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        bool ok;
        kp[t] = at(16 * t + lq, K, ok);
      }
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        bool ok;
        vp[e] = at(key_of(e, grp), V, ok);
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
    const bool fresh = j0 + KT > p.first;  // holds new rows, which not every row sees
    if (!all_there) {
#pragma unroll
      for (int e = 0; e < NV; ++e)
#pragma unroll
        for (int d = 0; d < DP; ++d) vv[e].v[d] = there >> e & 1u ? vv[e].v[d] : (T)0.f;
    }
    if (fresh) {
      const bool odd = take_out(vv, j0 - p.first, grp);
      dirty = dirty || odd;
    }
    float s[MT][NV];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t seen = there;
      if (fresh) seen = seen_keys<NV>(a, Query(a, p, qm[mt]), j0, p.first, grp, there);
      score_tile<T, D>(kv, qv[mt], !all_there || fresh, seen, s[mt]);
      run[mt].weigh(s[mt], a.scale2);
    }
    add_values<T, D, MT, MT == 1 || is_prefix<A>>(vv, s, run);
  }

  // the join: 16 rows at a time; thread -> row tid / 16, elements DP (tid % 16) ..
  if (dirty && lane == 0) atomicOr(&s_dirty, 1);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float ls = run[mt].sum();
    if (mt) __syncthreads();
    if (grp == 0) sML[wave][lq] = make_float2(run[mt].mx, ls);
#pragma unroll
    for (int d = 0; d < DP; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) sO[wave][lq][D / 4 * grp + DP * r + d] = run[mt].o[d][r];
    __syncthreads();
    const int row16 = tid >> 4, d0 = DP * (tid & 15), m = p.m0 + 16 * mt + row16;
    if (m < p.mrows) {
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
      const Query x(a, p, m);
      if (s_dirty) put_back<T, D>(a, p, x, [&](const T* v) {
#pragma unroll
        for (int d = 0; d < DP; ++d) O[d] += taken_out(v[d0 + d]);
      });
      if (p.whole) {
        T* out = reinterpret_cast<T*>(a.out) + x.row * a.o_row + x.h * a.o_head + d0;
        Piece<T, DP> r;
#pragma unroll
        for (int d = 0; d < DP; ++d) r.v[d] = (T)(L == 0.f ? 0.f : O[d] / L);
        if (a.o_wide) {
          *reinterpret_cast<Piece<T, DP>*>(out) = r;
        } else {
#pragma unroll
          for (int d = 0; d < DP; ++d) out[d] = r.v[d];
        }
      } else {
        const size_t at = slot_of(a, plan, p, (size_t)x.row * a.q_heads + x.h);
#pragma unroll
        for (int d = 0; d < DP; ++d) part.o[at * D + d0 + d] = O[d];
        if ((tid & 15) == 0) part.ml[at] = make_float2(mm, L);
      }
      if ((tid & 15) == 0) tell_parts(a, plan, p, part, (size_t)x.row * a.q_heads + x.h);
    }
  }
}

// s_waitcnt vmcnt(N), the other counts left alone.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
// Every wave's LDS reads are done and its loads as far as it waited for: a
// barrier without the wait for all loads that __syncthreads adds.
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0)
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __asm__ volatile("" ::: "memory");
}
// Each lane's 16 bytes at its own address to lds + 16 * lane (lds the same for
// the wave), without registers.
__device__ __forceinline__ void load_to_lds(const void* src, lds_ptr_t* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, lds, 16, 0, 0);
#endif
}
// Each lane's 4 bytes to lds + 4 * lane.
__device__ __forceinline__ void load4_to_lds(const void* src, lds_ptr_t* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, lds, 4, 0, 0);
#endif
}

// Many query rows: the block's waves have 16 WMT of them each and go over the
// split's keys together, 16 KB of keys and values at a time.  Those are read
// once for wide_rows of queries.  A ring of three buffers in LDS is filled by direct
// loads, two buffers ahead (one ahead, through registers, each of them was
// waited for: about 2 us a buffer).  16-byte places of a row are exchanged by XOR
// with the row's number, so that 16 rows' same place are read at once.
//
// Where all blocks have as many keys it is bound by the SIMDs' issue: 63 rows of 32 query
// heads on 8 of 128 over 65536 f16 keys take 102 us (665 TFLOP/s; 1.5 us a buffer of 32
// keys of a CU's two blocks), of whose SIMD cycles 56% are vector instructions (the
// weights: an exponential, a conversion and a move into the operand of each score) and
// 38% matrix ones, which hardly overlap.  fp32, 100 rows of 20 heads of 64 over 8000
// keys, 65 us: 24% and 72%.  Batches lose to their raggedness: blocks have the longest
// sequence's keys, 33 buffers in 57 us for trees of up to 63 rows over up to 4099 f16
// keys, where an even share is 22.8, and 23% of the tiles' rows are none; chains of 257
// and 180 rows over 1201 and 841 fp32 keys 10 buffers in 41 us, an even share 6.6.  A ring
// of five buffers was 2.5% faster on the trees and leaves no LDS, two buffers of
// twice the keys, with half the barriers, as fast.
//
// The ring's buffers are objects of their own, named by constants in the usual
// path: a read that might alias any of them would wait for every load.
template <typename T, int D, typename A>
__global__ __launch_bounds__(kAttendThreads, wide_blocks<A>) void attend_wide_kernel(A a, AttendPlan plan, Parts part) {
  typedef Dims<T, D> S;
  typedef typename Mat<T>::op Op;
  constexpr int KT = S::KT, NT = S::NT, DP = S::DP, DC = S::DC, NV = S::NV;
  constexpr int E16 = 16 / sizeof(T);             // elements of 16 bytes
  constexpr int CPR = D / E16;                    // 16-byte places of a row
  constexpr int KEYS = 512 / CPR;                 // keys of a buffer: 8 KB each of keys and values
  constexpr int STEP = kAttendThreads / CPR;      // rows a pass of the block loads
  constexpr int PASSES = KEYS / STEP;             // 2
  constexpr int WMT = (is_prefix<A> ? kPrefixRows : wide_rows(sizeof(T) == 4)) / (16 * kAttendWaves);
  constexpr int XM = CPR < 16 ? CPR - 1 : 15;
  constexpr bool WHOLE = is_prefix<A> && sizeof(T) == 2;
  __shared__ __attribute__((aligned(1024))) u32x4 sK0[KEYS * CPR], sK1[KEYS * CPR], sK2[KEYS * CPR];
  __shared__ __attribute__((aligned(1024))) u32x4 sV0[KEYS * CPR], sV1[KEYS * CPR], sV2[KEYS * CPR];
  auto bufK = [&](int b) -> u32x4* { return b == 0 ? sK0 : b == 1 ? sK1 : sK2; };
  auto bufV = [&](int b) -> u32x4* { return b == 0 ? sV0 : b == 1 ? sV1 : sV2; };

  Part p;
  if (!find_part(a, plan, 16 * WMT * kAttendWaves, p)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 15, grp = lane >> 4;
  const int wm0 = p.m0 + 16 * WMT * wave;
  const bool works = wm0 < p.mrows;
  if (!a.mask) {  // a chain: nobody sees past the block's last row
    const Query x(a, p, min(p.m0 + 16 * WMT * kAttendWaves, p.mrows) - 1);
    p.end = min(p.end, max(p.first + x.i + 1, p.begin));
  }
  const Query last_q(a, p, min(wm0 + 16 * WMT, p.mrows) - 1);
  // Keys before this one are seen by all of the wave's rows: of a chain's new rows
  // those up to the wave's first.
  const int open = a.mask ? p.first : p.first + Query(a, p, min(wm0, p.mrows - 1)).i + 1;

  // This thread's rows of a buffer, and its place of them.
  const int row0 = tid / CPR;
  const int64_t head = p.kvh * a.c.head_stride(D);
  const T* K = reinterpret_cast<const T*>(a.c.k) + head;
  const T* V = reinterpret_cast<const T*>(a.c.v) + head;
  const int32_t* table = a.c.table + (size_t)p.seq * a.c.table_stride;
  // The lanes hold 64 of the sequence's table entries, from number `held` on; a
  // row's comes by a shuffle.  (Looked up a buffer ahead, each wait for one
  // waited for the loads in flight as well.)
  int held = INT_MIN, entries = 0;
  const bool in_a_page = (1 << a.c.page_shift) >= KEYS;  // (buffers start at multiples of KEYS)
  uint32_t mine[PASSES];  // this thread's elements of a buffer that lies in one page
#pragma unroll
  for (int u = 0; u < PASSES; ++u) mine[u] = (row0 + STEP * u) * D + ((tid % CPR) ^ ((row0 + STEP * u) & XM)) * E16;
  auto entry_of = [&](int j) { return __shfl(entries, (j >> a.c.page_shift) - held, kWave); };
  // Starts a buffer's loads (rows that are not there read page 0); which keys are
  // there, as bits (lanes past KEYS repeat).
  auto load = [&](int j0, int buf) {
    const int at0 = min(j0, p.len - 1);
    if (held < 0 || (min(at0 + KEYS, p.len) - 1) >> a.c.page_shift >= held + 64) {
      held = at0 >> a.c.page_shift;
      entries = table[min(held + lane, (p.len - 1) >> a.c.page_shift)];
      __asm__ volatile("" : "+v"(entries));  // (waits here, not wherever it is used)
    }
    u32x4 *k = bufK(buf) + 64 * wave, *v = bufV(buf) + 64 * wave;
    const int j = j0 + (lane & (KEYS - 1));
    if (in_a_page) {  // one entry for all, and only the page differs from buffer to buffer
      const int entry = __builtin_amdgcn_readlane(entries, (at0 >> a.c.page_shift) - held);
      const bool ok = (unsigned)entry < (unsigned)a.c.pages;
      const int64_t page = a.c.row_in(ok ? entry : 0, j0, D);
#pragma unroll
      for (int u = 0; u < PASSES; ++u) {
        load_to_lds(K + page + mine[u], (lds_ptr_t*)(k + kAttendThreads * u));
        load_to_lds(V + page + mine[u], (lds_ptr_t*)(v + kAttendThreads * u));
      }
      return (uint64_t)__ballot(ok && j < p.len);
    }
#pragma unroll
    for (int u = 0; u < PASSES; ++u) {
      const int r = row0 + STEP * u;
      const int page = entry_of(min(j0 + r, p.len - 1));
      const int64_t at = a.c.row_in((unsigned)page < (unsigned)a.c.pages ? page : 0, j0 + r, D) + ((tid % CPR) ^ (r & XM)) * E16;
      load_to_lds(K + at, (lds_ptr_t*)(k + kAttendThreads * u));
      load_to_lds(V + at, (lds_ptr_t*)(v + kAttendThreads * u));
    }
    return (uint64_t)__ballot((unsigned)entry_of(min(j, p.len - 1)) < (unsigned)a.c.pages && j < p.len);
  };

  int qm[WMT];
  Op qv[WMT][DC];
  Running<T, D> run[WMT];
#pragma unroll
  for (int mt = 0; mt < WMT; ++mt) {
    qm[mt] = min(wm0 + 16 * mt + lq, p.mrows - 1);
    load_query<T, D>(a, Query(a, p, qm[mt]), grp, qv[mt]);
    run[mt].clear();
  }

  // The keys that are there, of this buffer, the next and the one after.
  constexpr uint64_t all_keys = ~0ull;
  uint64_t there0 = 0, there1 = 0, there2 = 0;
  if (p.begin < p.end) {
    there0 = load(p.begin, 0);
    there1 = load(p.begin + KEYS, 1);
    there2 = load(p.begin + 2 * KEYS, 2);
    wait_loads<4 * PASSES>();
    meet();
  }

  // A tile's keys and values from a buffer.  Of the places that a lane reads, those
  // of other rows are constants away, and those of other pieces of a row are an
  // XOR of the number's low bits.  The empty statement keeps the compiler
  // from holding each such address for each buffer throughout (about 100 registers).
  const int k_place = lq * CPR + ((sizeof(T) == 2 ? grp : DC / 4 * grp) ^ (lq & XM));
  constexpr int PB = DP * sizeof(T), PV = PB <= 16 ? 1 : PB / 16;  // bytes of a lane's piece of a value, 16-byte places
  const int v_place = (4 * grp * CPR + ((lq * PB / 16) ^ (4 * grp & XM))) * 16 + (PB < 16 ? lq * PB % 16 : 0);
  auto read_keys = [&](const u32x4* tk, Op(&kv)[NT][DC]) {
    int at = k_place;
    __asm__ volatile("" : "+v"(at));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int c = 0; c < DC; ++c) kv[t][c] = *reinterpret_cast<const Op*>(&tk[(at ^ 4 * c) + 16 * t * CPR]);
      } else {
#pragma unroll
        for (int c = 0; c < DC; c += 4) {
          const floatx4 x = *reinterpret_cast<const floatx4*>(&tk[(at ^ c / 4) + 16 * t * CPR]);
          kv[t][c] = x[0]; kv[t][c + 1] = x[1]; kv[t][c + 2] = x[2]; kv[t][c + 3] = x[3];
        }
      }
    }
  };
  auto read_values = [&](const u32x4* tv, Piece<T, DP>(&vv)[NV]) {
    int at = v_place;
    __asm__ volatile("" : "+v"(at));
    const char* base = reinterpret_cast<const char*>(tv);
#pragma unroll
    for (int e = 0; e < NV; ++e) {
      const int row = (16 * (e >> 2) + (e & 3)) * CPR * 16;
#pragma unroll
      for (int u = 0; u < PV; ++u) {
        const Piece<T, DP / PV> x = *reinterpret_cast<const Piece<T, DP / PV>*>(base + (at ^ ((e & 3) ^ u) * 16) + row);
#pragma unroll
        for (int d = 0; d < DP / PV; ++d) vv[e].v[u * (DP / PV) + d] = x.v[d];
      }
    }
  };
  // This buffer is read, by every wave, and the next has landed; the one after the
  // two to come is filled in its place.
  auto advance = [&](int buf, int& b0) {
    wait_loads<2 * PASSES>();
    meet();
    there0 = there1;
    there1 = there2;
    there2 = load(b0 + 3 * KEYS, buf);
    b0 += KEYS;
  };

  // All rows see all keys of the buffers up to the first that holds a row which
  // not all see, or misses one: a loop of its own, whose turns follow each other without a branch
  // that could meet the outputs' registers (merged, they were kept twice).  A tile's
  // values are on their way during its weights, the next tile's keys during its
  // second products.
  int b0 = p.begin, buf = 0;
  if (works) {
    auto plain = [&] { return there0 == all_keys && b0 + KEYS <= open && b0 < p.end; };
    Op kv[NT][DC];
    if (plain()) read_keys(bufK(0), kv);
    auto one = [&](auto buf_) {
      constexpr int B = decltype(buf_)::value, TILES = KEYS / KT;
#pragma unroll
      for (int sub = 0; sub < TILES; ++sub) {
        float s[WMT][NV];
        Piece<T, DP> vv[NV];
#pragma unroll
        for (int mt = 0; mt < WMT; ++mt) score_tile<T, D>(kv, qv[mt], false, 0u, s[mt]);
        __builtin_amdgcn_s_setprio(0);
        read_values(bufV(B) + sub * KT * CPR, vv);
#pragma unroll
        for (int mt = 0; mt < WMT; ++mt) run[mt].weigh(s[mt], a.scale2);
        if (sub + 1 < TILES) {
          read_keys(bufK(B) + (sub + 1) * KT * CPR, kv);
        } else {
          advance(B, b0);
          read_keys(bufK(B == 2 ? 0 : B + 1), kv);
        }
        __builtin_amdgcn_s_setprio(1);
        add_values<T, D, WMT, WHOLE, false>(vv, s, run);
      }
    };
    for (;;) {
      buf = 0;
      if (!plain()) break;
      one(std::integral_constant<int, 0>{});
      buf = 1;
      if (!plain()) break;
      one(std::integral_constant<int, 1>{});
      buf = 2;
      if (!plain()) break;
      one(std::integral_constant<int, 2>{});
    }
  }
  const int all_see = b0;
  // The other buffers: keys may be missing or new, so that not all rows see them all
  // (query tiles one after the other, for fewer registers).
  bool dirty = false;
  auto rest = [&](int j0, uint32_t bits, const u32x4* tk, const u32x4* tv) {
    // (past the end, or past what a chain's rows of this wave see)
    if (j0 >= p.end || (!a.mask && j0 - p.first > last_q.i)) return;
    bits >>= 4 * grp;
    const uint32_t there = NT == 2 ? (bits & 15u) | (bits >> 12 & 0xf0u) : bits & 15u;
#pragma unroll
    for (int mt = 0; mt < WMT; ++mt) {
      float s[1][NV];
      {
        Op kv[NT][DC];
        read_keys(tk, kv);
        int m = qm[mt];
        __asm__ volatile("" : "+v"(m));
        const uint32_t seen = seen_keys<NV>(a, Query(a, p, m), j0, p.first, grp, there);
        score_tile<T, D>(kv, qv[mt], true, seen, s[0]);
      }
      Piece<T, DP> vv[NV];
      read_values(tv, vv);
#pragma unroll
      for (int e = 0; e < NV; ++e)
#pragma unroll
        for (int d = 0; d < DP; ++d) vv[e].v[d] = there >> e & 1u ? vv[e].v[d] : (T)0.f;
      if (j0 + KT > p.first) {
        const bool odd = take_out(vv, j0 - p.first, grp);
        dirty = dirty || odd;
      }
      run[mt].weigh(s[0], a.scale2);
      add_values<T, D, 1, WHOLE, false>(vv, s, run + mt);
    }
  };
  for (; b0 < p.end; buf = buf == 2 ? 0 : buf + 1) {
    if (works)
#pragma unroll 1
      for (int sub = 0; sub < KEYS / KT; ++sub)
        rest(b0 + sub * KT, (uint32_t)(there0 >> (sub * KT)), bufK(buf) + sub * KT * CPR, bufV(buf) + sub * KT * CPR);
    advance(buf, b0);
  }
  wait_loads<0>();  // (LDS must not be written after the block's end)

#pragma unroll
  for (int mt = 0; mt < WMT; ++mt) {
    const float L = run[mt].sum();
    if (WHOLE) infinities<T, D>(a, p, min(p.end, max(p.first, all_see)), run[mt].o, L);
    if (wm0 + 16 * mt + lq >= p.mrows) continue;
    const Query x(a, p, qm[mt]);
    const int d0 = D / 4 * grp;
    if (dirty) put_back<T, D>(a, p, x, [&](const T* v) {
#pragma unroll
      for (int d = 0; d < DP; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) run[mt].o[d][r] += taken_out(v[d0 + DP * r + d]);
    });
    if (p.whole) {
      T* out = reinterpret_cast<T*>(a.out) + x.row * a.o_row + x.h * a.o_head + d0;
      const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        Piece<T, DP> y;
#pragma unroll
        for (int d = 0; d < DP; ++d) y.v[d] = (T)(L == 0.f ? 0.f : run[mt].o[d][r] * inv);
        if (a.o_wide) {
          *reinterpret_cast<Piece<T, DP>*>(out + DP * r) = y;
        } else {
#pragma unroll
          for (int d = 0; d < DP; ++d) out[DP * r + d] = y.v[d];
        }
      }
    } else {
      const size_t at = slot_of(a, plan, p, (size_t)x.row * a.q_heads + x.h);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d = 0; d < DP; d += 4)
          *reinterpret_cast<floatx4*>(part.o + at * D + d0 + DP * r + d) =
              floatx4{run[mt].o[d][r], run[mt].o[d + 1][r], run[mt].o[d + 2][r], run[mt].o[d + 3][r]};
      if (grp == 0) part.ml[at] = make_float2(run[mt].mx, L);
    }
    if (grp == 0) tell_parts(a, plan, p, part, (size_t)x.row * a.q_heads + x.h);
  }
}

// Joins a row and query head's splits, WAVES waves for each: lane groups of D/4
// take every so manyth split, four elements a lane.  One wave where there are
// at most kFewSplits: blocks of a wave each then fill the chip with less, and
// each asks for all it may need at once (what its loads wait for is most of its
// time: 3.0 us with the row's sequence looked up first, 2.1 so).
constexpr int kFewSplits = 16, kMaxSplits = 256;
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void combine_kernel(AttendArgs a, AttendPlan plan, Parts part) {
  constexpr int L4 = D / 4, G = WAVES * 64 / L4;
  constexpr int AHEAD = (kFewSplits + G - 1) / G;  // loads of a lane ahead of the weights
  __shared__ floatx4 sO[G][L4];
  __shared__ float sF[kMaxSplits], sW[WAVES], sL[WAVES];
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const size_t pair = (size_t)row * a.q_heads + h, at = pair * plan.splits;
  const int g = tid / L4, l4 = tid - g * L4;
  const floatx4* po = reinterpret_cast<const floatx4*>(part.o + at * D) + l4;
  const int n = min(part.n[pair], plan.splits);  // (splits the row has)
  const bool mine = row >= a.r.start[0] && row < a.r.start[a.r.seqs];
  float2 ml = tid < plan.splits ? part.ml[at + tid] : make_float2(-INFINITY, 0.f);
  floatx4 x[AHEAD];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) x[u] = po[(size_t)min(g + u * G, plan.splits - 1) * L4];
  if (!mine || n <= 1) return;  // nobody's row, or final already
  if (tid >= n) ml = make_float2(-INFINITY, 0.f);
  float mm = ml.x;
#pragma unroll
  for (int off = 32; off; off >>= 1) mm = fmaxf(mm, __shfl_xor(mm, off, kWave));
  if (WAVES > 1) {
    if ((tid & 63) == 0) sW[tid >> 6] = mm;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) mm = fmaxf(mm, sW[w]);
  }
  const float base = mm == -INFINITY ? 0.f : mm;
  const float f = exp2f(ml.x - base);
  sF[tid] = f;
  float L = warp_sum(f * ml.y);
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
#pragma unroll 4
    for (int s = g + AHEAD * G; s < n; s += G) O += sF[s] * po[(size_t)s * L4];
    sO[g][l4] = O;
  }
  __syncthreads();
  if (tid >= L4) return;
  floatx4 O = sO[0][tid];
#pragma unroll
  for (int w = 1; w < G; ++w) O += sO[w][tid];
  const float inv = 1.f / L;
  T* out = reinterpret_cast<T*>(a.out) + row * a.o_row + h * a.o_head + 4 * tid;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(L == 0.f ? 0.f : O[e] * inv);
}

void attend_launched(hipError_t e);  // throws HipError (kv_ops.hip)

// The launch of a plan's blocks.
template <typename T, int D, typename A>
void launch_tiles(const A& a, const AttendPlan& plan, const Parts& part, AttendGrid g, hipStream_t s) {
  const dim3 grid(g.x, g.y), block(kAttendThreads);
  const bool big = (1 << a.c.page_shift) >= Mat<T>::KT;
  auto tiles = [&](auto big_page) {
    constexpr bool BIG = decltype(big_page)::value;
    if (plan.form == 1)
      hipLaunchKernelGGL((attend_kernel<T, D, 1, BIG, A>), grid, block, 0, s, a, plan, part);
    else
      hipLaunchKernelGGL((attend_kernel<T, D, 2, BIG, A>), grid, block, 0, s, a, plan, part);
  };
  if (plan.form == kWide) {
    if constexpr (wide_dim(D)) hipLaunchKernelGGL((attend_wide_kernel<T, D, A>), grid, block, 0, s, a, plan, part);
  } else if (big) {
    tiles(std::true_type{});
  } else {
    tiles(std::false_type{});
  }
  attend_launched(hipGetLastError());
}

template <typename T, int D>
void launch_attend(const AttendArgs& a, const AttendPlan& plan, void* workspace, hipStream_t s) {
  const size_t pairs = (size_t)a.r.rows * a.q_heads, n = pairs * plan.splits;
  Parts part;
  part.o = static_cast<float*>(workspace);
  part.ml = reinterpret_cast<float2*>(part.o + n * D);
  part.n = reinterpret_cast<int32_t*>(part.ml + n);
  launch_tiles<T, D>(a, plan, part, attend_grid(plan, a.c.kv_heads), s);
  if (plan.splits == 1) return;
  if (plan.splits <= kFewSplits)
    hipLaunchKernelGGL((combine_kernel<T, D, 1>), dim3(a.r.rows, a.q_heads), dim3(64), 0, s, a, plan, part);
  else
    hipLaunchKernelGGL((combine_kernel<T, D, 4>), dim3(a.r.rows, a.q_heads), dim3(256), 0, s, a, plan, part);
  attend_launched(hipGetLastError());
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

#endif  // KV_ATTEND_KERNELS

}  // namespace mit2hip
