// kv_evict.hip -- rows of least weight leave a paged cache (see kv_ops.h and
// mit2cfm.h for what it computes).
#include <algorithm>
#include <type_traits>

#include "kv_args.h"

namespace mit2hip {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kKeys = 16;                         // a thread's keys at a time
constexpr int kWaveKeys = 64 * kKeys;             // a wave's
constexpr int kSplitThreads = 512, kSplitWaves = kSplitThreads / 64;
constexpr int kSplitKeys = kSplitWaves * kWaveKeys;  // a segment's, where the length is as said
constexpr int kBins = 2048;
constexpr int kMaxSegments = 64;
// Rows that leave a line of one wave are found one after the other up to this many: 1440
// lines of 704 places, with the moves, on the same data again and again, 10.7, 11.5, 12.8, 16.0,
// 18.5 us for 1, 2, 4, 8, 12 rows, by the search 16.2 to 18.6 (one row 18.9).
constexpr int kFewLeave = 8;
constexpr int kMoveThreads = 256, kMoveBatch = 2;  // a thread's moves in flight

struct EvictArgs {
  CacheView c;
  const int32_t *length, *keep;
  const float* weights;
  float* weights_out;
  const int32_t *born, *now;
  int32_t *born_out, *length_out;
  int64_t stride;   // of a line: a layer's, sequence's and key head's weights
  int64_t layer16;  // 16-byte vectors from a layer's k (v) to the next's
  int row16;        // of a row
  int seqs;
  int64_t first_rows, last_rows;
  // workspace: a line's list of moves (places that rows left, places they come
  // from: list_stride of each), their number, a sequence's new length
  int32_t *to, *from, *moves, *stay;
  int64_t list_stride;
  // long lines: histograms [line][segment][kBins] of three rounds, and what they tell
  uint32_t* hist[3];
  uint2* found[2];  // [line] the bits so far, rows that stay among the keys that have them
  uint32_t* larger;  // [line][segment] keys above those that agree in the first two rounds' bits
  int segments;
};

__device__ __forceinline__ int64_t line_of(const EvictArgs& a, int layer, int seq, int head) {
  return ((int64_t)layer * a.seqs + seq) * a.c.kv_heads + head;
}
// Places of a sequence that count.
__device__ __forceinline__ int places_of(const EvictArgs& a, int seq) {
  return (int)min((int64_t)max(0, min(a.length[seq], a.c.capacity())), a.stride);
}

// What a line's places are ranked by: larger keys stay.  Protected places above all
// weights, NaN and places without a page below all.
struct Ranks {
  const float* weights;
  const int32_t* born;
  const int32_t* table;
  int n, first, tail, pages, page_shift;  // tail: the first of the youngest places, without births
  int oldest;                             // with births: rows from this one on
  __device__ __forceinline__ uint32_t key_of(int j, float weight, int birth, int page) const {
    const bool stays = (j < first) | (born ? birth >= oldest : j >= tail);
    uint32_t u = __float_as_uint(weight);
    u = u == 0x80000000u ? 0u : u;
    const bool least = ((u & 0x7fffffffu) > 0x7f800000u) | ((unsigned)page >= (unsigned)pages);
    u ^= u >> 31 ? 0xffffffffu : 0x80000000u;
    return stays ? 0xffffffffu : least ? 0u : u;
  }
  // The keys of a wave's places j0 .. j1 - 1 (at most kWaveKeys) to LDS, one after
  // the other, 0 past the end.  Read through resources that end where the places do.
  // then(place, weight, birth) of each place.
  template <typename F>
  __device__ __forceinline__ void load(int j0, int j1, uint32_t* to, F&& then) const {
    constexpr int B = kKeys;  // of a lane at once
    const int lane = threadIdx.x & 63, size = max(j1 - j0, 0);
    const int e0 = j0 >> page_shift, entries = size ? ((j1 - 1) >> page_shift) - e0 + 1 : 0;
    const buffer_rsrc_t rw = make_buffer_rsrc(weights + j0, 4 * size), rt = make_buffer_rsrc(table + e0, 4 * entries);
    const buffer_rsrc_t rb = make_buffer_rsrc(born ? born + j0 : nullptr, born ? 4 * size : 0);
#pragma unroll 1
    for (int i0 = 0; i0 < kWaveKeys; i0 += 64 * B) {
      float w[B];
      int birth[B], page[B];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const int i = i0 + 64 * u + lane;
        w[u] = buffer_load_f32(rw, 4 * i);
        birth[u] = __float_as_int(buffer_load_f32(rb, 4 * i));
        page[u] = __float_as_int(buffer_load_f32(rt, 4 * (((j0 + i) >> page_shift) - e0)));
      }
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const int i = i0 + 64 * u + lane;
        to[i] = i < size ? key_of(j0 + i, w[u], birth[u], page[u]) : 0u;
        if (i < size) then(j0 + i, w[u], birth[u]);
      }
    }
  }
};

// count += key >= least, in two instructions (compiled, it was a select and a sum besides the comparison).
__device__ __forceinline__ void add_if_from(uint32_t& count, uint32_t key, uint32_t least) {
#if defined(__HIP_DEVICE_COMPILE__)
  __asm__("v_cmp_le_u32 vcc, %1, %2\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc" : "+v"(count) : "s"(least), "v"(key) : "vcc");
#else
  count += key >= least;
#endif
}
// The sum over a wave, in all lanes.
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#if defined(__HIP_DEVICE_COMPILE__)
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1 .. 8: a row's sum in its last lane
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15, to the rows after the first and third
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return __builtin_amdgcn_readlane(v, 63);
#else
  return v;
#endif
}
// The least (the largest) over a wave, in all lanes.
template <bool LEAST>
__device__ __forceinline__ uint32_t wave_end(uint32_t v) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr uint32_t none = LEAST ? 0xffffffffu : 0u;
  auto join = [&](uint32_t o) { v = LEAST ? min(v, o) : max(v, o); };
  join(__builtin_amdgcn_update_dpp(none, v, 0x111, 0xf, 0xf, false));
  join(__builtin_amdgcn_update_dpp(none, v, 0x112, 0xf, 0xf, false));
  join(__builtin_amdgcn_update_dpp(none, v, 0x114, 0xf, 0xf, false));
  join(__builtin_amdgcn_update_dpp(none, v, 0x118, 0xf, 0xf, false));
  join(__builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false));
  join(__builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
#else
  return v;
#endif
}
// base + #(voting lanes before this one)
__device__ __forceinline__ uint32_t lanes_below(uint64_t vote, uint32_t base) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(vote >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)vote, base));
}
// An element at a 32-bit distance in bytes.
template <typename T>
__device__ __forceinline__ T& near(T* base, uint32_t i) {
  return *reinterpret_cast<T*>(reinterpret_cast<std::conditional_t<std::is_const<T>::value, const char, char>*>(base) + (uint32_t)(4u * i));
}

// A line as its block sees it.
struct Line {
  int head, seq, layer;
  int64_t at;
  int m;  // rows that stay
  bool apart, apart_born;
  float* weights_out;
  int32_t* born_out;
  Ranks r;
  __device__ __forceinline__ Line(const EvictArgs& a, int head_) : head(head_), seq(blockIdx.y), layer(blockIdx.z) {
    at = line_of(a, layer, seq, head);
    r.n = places_of(a, seq);
    m = min(r.n, max(a.keep[seq], 0));
    apart = a.weights_out != a.weights;
    apart_born = a.born && a.born_out != a.born;
    r.weights = a.weights + at * a.stride;
    r.born = a.born ? a.born + at * a.stride : nullptr;
    r.table = a.c.table + (size_t)seq * a.c.table_stride;
    r.first = (int)min(a.first_rows, (int64_t)r.n);
    r.tail = (int)max(r.n - a.last_rows, (int64_t)0);
    r.pages = a.c.pages;
    r.page_shift = a.c.page_shift;
    r.oldest = a.born ? (int)max((int64_t)a.now[seq] - a.last_rows, (int64_t)INT32_MIN) : 0;
    weights_out = a.weights_out + at * a.stride;
    born_out = a.born_out ? a.born_out + at * a.stride : nullptr;
  }
  // A wave's keys to LDS (Ranks::load), the weights and births below m to where they are
  // wanted.  (Those of places that rows left are written again by the moves.)
  __device__ __forceinline__ void load(int j0, int j1, uint32_t* to) const {
    r.load(j0, j1, to, [&](int j, float weight, int birth) {
      if (apart && j < m) near(weights_out, j) = weight;
      if (apart_born && j < m) near(born_out, j) = birth;
    });
  }
  // Those of the places j0 .. j1 - 1 below m, by `by` threads.
  __device__ __forceinline__ void copy(int j0, int j1, int mine, int by) const {
    if (!apart && !apart_born) return;
    constexpr int B = 8;  // of a thread in flight
    j1 = min(j1, m);
#pragma unroll 1
    for (int j = j0 + mine; j < j1; j += B * by) {
      float w[B];
      int birth[B];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const int at = min(j + u * by, j1 - 1);
        if (apart) w[u] = near(r.weights, at);
        if (apart_born) birth[u] = near(r.born, at);
      }
#pragma unroll
      for (int u = 0; u < B; ++u)
        if (j + u * by < j1) {
          if (apart) near(weights_out, j + u * by) = w[u];
          if (apart_born) near(born_out, j + u * by) = birth[u];
        }
    }
  }
};

// A wave's places j0 .. j1 - 1 in order, 64 at a time: f(place, key, whether it is one of
// them).  held: `keys` has them; else it is filled as they come.
template <typename F>
__device__ __forceinline__ void sweep(const Ranks& r, int j0, int j1, bool held, uint32_t* keys, F&& f) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int base = j0; base < j1; base += kWaveKeys) {
    const int size = min(j1 - base, kWaveKeys);
    if (!held) r.load(base, base + size, keys, [](int, float, int) {});
#pragma unroll 1
    for (int i = lane; i - lane < size; i += 256) {  // (four at once wait once; past the end they count for nothing)
      uint32_t k[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) k[u] = keys[i + 64 * u];
#pragma unroll
      for (int u = 0; u < 4; ++u) f(base + i + 64 * u, k[u], i + 64 * u < size);
    }
  }
}

// Writes the lists' share of a wave's places.  Keys above `least` stay, and the first
// `ties` that equal it.  A place p that stays has before(p) = #(larger keys before p) +
// min(#(equal keys before p), ties) rows before it that stay, which gives a freed place
// and a row that moves their numbers in the lists: p - before(p), before(p) - stay_below.
// gt, eq: larger and equal keys of the places before the wave's.
__device__ __forceinline__ void list_moves(const EvictArgs& a, const Line& x, int j0, int j1, bool held, uint32_t* keys,
                                           uint32_t least, uint32_t ties, uint32_t gt, uint32_t eq, uint32_t stay_below) {
  int32_t *to = a.to + x.at * a.list_stride, *from = a.from + x.at * a.list_stride;
  sweep(x.r, j0, j1, held, keys, [&](int j, uint32_t k, bool in) {
    const bool more = in && k > least, equal = in && k == least;
    const uint64_t vote_gt = __ballot(more), vote_eq = __ballot(equal);
    const uint32_t gt_before = lanes_below(vote_gt, gt), eq_before = lanes_below(vote_eq, eq);
    const uint32_t before = gt_before + min(eq_before, ties);
    const bool stays = more || (equal && eq_before < ties);
    if (j < x.m) {
      if (in && !stays) near(to, j - before) = j;
    } else if (stays) {
      near(from, before - stay_below) = j;
    }
    gt += __popcll(vote_gt);
    eq += __popcll(vote_eq);
  });
}

// A block of W waves ranks a line whose keys lie in registers (longer lines than were
// said are read again each time).  The key of the last row that stays, the m-th
// largest, is found from the top, by one wave a bit at a time, by more, which wait for
// each other at every step, two: the lanes count the keys from one candidate, or each of
// three, on, and the search ends once these are m.  No histogram, so no addition waits
// for another, and of one wave no barrier.
//
// Instructions and waits bound it, not its few bytes.  1440 lines of 703 of 704 places, one
// wave each: 7 us (13.5 by the search); 256 lines of 8191, eight waves:
// 22 us.  More waves for a line wait longer for each other than they count less: lines of
// 1000 (32 of them, with the moves) 15.7, 18.4, 20.4 us by 1, 4, 8 waves, of 4000 22.8, 24.5,
// 40.2 by 4, 8, 16, of 8000 29.2 and 48.4 by 8 and 16.
template <int W>
__global__ __launch_bounds__(64 * W) void choose_kernel(EvictArgs a) {
  __shared__ uint32_t s_keys[W][kWaveKeys];
  constexpr int BITS = W == 1 ? 1 : 2, N = (1 << BITS) - 1;  // of a step, and its candidates
  __shared__ uint2 s_count[2][W];
  __shared__ uint32_t s_gt[W], s_eq[W], s_gt_below[W], s_eq_below[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Line x(a, blockIdx.x);
  const int n = x.r.n, m = x.m;
  if (tid == 0 && x.head == 0 && x.layer == 0) a.stay[x.seq] = m;
  if (m == n || m == 0) {
    if (tid == 0) a.moves[x.at] = 0;
    x.copy(0, m, tid, 64 * W);
    return;
  }
  const bool held = n <= W * kWaveKeys;
  const int share = held ? kWaveKeys : ((n + W - 1) / W + 63) / 64 * 64;  // a wave's places
  const int j0 = min(wave * share, n), j1 = min(j0 + share, n);
  uint32_t* const keys = s_keys[wave];
  uint32_t key[kKeys];
  if (held) {
    x.load(j0, j1, keys);
#pragma unroll
    for (int i = 0; i < kKeys; ++i) key[i] = keys[64 * i + lane];
  }

  // Few rows leave: the last of the least, as often as that, and the rows behind the budget
  // that are not of them take their places.
  if (held && n - m <= (W == 1 ? kFewLeave : 1)) {
    uint32_t taken = 0;  // of this lane's keys, a bit each
    auto last_of_least = [&]() {
      uint32_t low = 0xffffffffu, place = 0;
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
        if (j0 + 64 * i + lane < j1 && key[i] <= low && !(taken >> i & 1u)) {
          low = key[i];
          place = j0 + 64 * i + lane;
        }
      const uint32_t least = wave_end<true>(low);
      return make_uint2(least, wave_end<false>(low == least ? place : 0u));
    };
    int32_t *const to = a.to + x.at * a.list_stride, *const from = a.from + x.at * a.list_stride;
    if constexpr (W == 1) {
      const int leave = n - m;
      uint32_t gone = 0, mine = 0xffffffffu;  // of the rows from m on, a bit each; of the leaving ones, lane by lane
#pragma unroll 1
      for (int t = 0; t < leave; ++t) {
        const uint32_t place = last_of_least().y;
        if ((place & 63) == lane) taken |= 1u << (place >> 6);
        if (lane == t) mine = place;
        if (place >= (uint32_t)m) gone |= 1u << (place - m);
      }
      uint32_t before = 0;  // freed places before this lane's
#pragma unroll 1
      for (int t = 0; t < leave && leave > 1; ++t) before += __builtin_amdgcn_readlane(mine, t) < mine;
      if (mine < (uint32_t)m) to[before] = mine;
      if (lane < leave && !(gone >> lane & 1u)) from[__popc(~gone & ((1u << lane) - 1u))] = m + lane;
      if (lane == 0) a.moves[x.at] = leave - __popc(gone);
    } else {
      uint2 out = last_of_least();
      if (lane == 0) s_count[0][wave] = out;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < W; ++w) {  // (a wave without places tells of the largest key at the first)
          const uint2 o = s_count[0][w];
          if (o.x < out.x || (o.x == out.x && o.y > out.y)) out = o;
        }
        const bool moves = out.y < (uint32_t)m;
        a.moves[x.at] = moves;
        if (moves) {
          to[0] = out.y;
          from[0] = m;
        }
      }
    }
    return;
  }

  int turn = 0;
  // A lane's counts, over the block.
  auto whole = [&](uint32_t(&count)[N]) {
    if constexpr (N == 1) {
      count[0] = wave_sum(count[0]);
    } else {
      const uint32_t two = wave_sum(count[0] | count[1] << 16), third = wave_sum(count[2]);  // (at most 1024 of a wave)
      if (lane == 0) s_count[turn][wave] = make_uint2(two, third);
      __syncthreads();
      count[0] = count[1] = count[2] = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint2 o = s_count[turn][w];
        count[0] += o.x & 0xffffu;
        count[1] += o.x >> 16;
        count[2] += o.y;
      }
      turn ^= 1;
#pragma unroll
      for (int u = 0; u < 3; ++u) count[u] = __builtin_amdgcn_readfirstlane(count[u]);
    }
  };
  // Keys >= c[u]; c > 0, so none past the end.
  auto from_on = [&](const uint32_t(&c)[N], uint32_t(&count)[N]) {
#pragma unroll
    for (int u = 0; u < N; ++u) count[u] = 0;
    if (held) {
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
#pragma unroll
        for (int u = 0; u < N; ++u) add_if_from(count[u], key[i], c[u]);
      whole(count);
      return;
    }
    sweep(x.r, j0, j1, false, keys, [&](int, uint32_t k, bool) {
#pragma unroll
      for (int u = 0; u < N; ++u) count[u] += __popcll(__ballot(k >= c[u]));
    });
    if (W == 1) return;
    for (int u = 0; u < N; ++u) {  // (counts past 16 bits)
      __syncthreads();
      if (lane == 0) s_gt[wave] = count[u];
      __syncthreads();
      count[u] = 0;
      for (int w = 0; w < W; ++w) count[u] += s_gt[w];
      count[u] = __builtin_amdgcn_readfirstlane(count[u]);
    }
    __syncthreads();
  };
  uint32_t least = 0, ties = 0, c[N], count[N];
  bool exact = false;
  for (int bit = 32 - BITS; bit >= 0 && !exact; bit -= BITS) {
#pragma unroll
    for (int u = 0; u < N; ++u) c[u] = least | (u + 1u) << bit;
    from_on(c, count);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (exact) continue;
      if (count[u] >= (uint32_t)m) least = c[u];
      exact = count[u] == (uint32_t)m;
    }
  }
  if (exact) {
    least -= 1;  // all from the candidate on stay
  } else if (least == 0xffffffffu) {
    ties = m;
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u) c[u] = least + 1;
    from_on(c, count);
    ties = m - count[0];
  }

  uint32_t gt = 0, eq = 0, gt_below = 0, eq_below = 0;
  if (held) {
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const int j = j0 + 64 * i + lane;
      const uint32_t more = key[i] > least ? 1u : 0u, equal = j < j1 && key[i] == least ? 1u : 0u;
      gt += more;
      eq += equal;
      gt_below += j < m ? more : 0u;
      eq_below += j < m ? equal : 0u;
    }
    const uint32_t all = wave_sum(gt | eq << 16), low = wave_sum(gt_below | eq_below << 16);
    gt = all & 0xffffu;
    eq = all >> 16;
    gt_below = low & 0xffffu;
    eq_below = low >> 16;
  } else {
    sweep(x.r, j0, j1, held, keys, [&](int j, uint32_t k, bool in) {
      const uint64_t more = __ballot(in && k > least), equal = __ballot(in && k == least), low = __ballot(j < m);
      gt += __popcll(more);
      eq += __popcll(equal);
      gt_below += __popcll(more & low);
      eq_below += __popcll(equal & low);
    });
  }
  if (W > 1) {
    if (lane == 0) {
      s_gt[wave] = gt;
      s_eq[wave] = eq;
      s_gt_below[wave] = gt_below;
      s_eq_below[wave] = eq_below;
    }
    __syncthreads();
    gt = eq = gt_below = eq_below = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      gt += w < wave ? s_gt[w] : 0;
      eq += w < wave ? s_eq[w] : 0;
      gt_below += s_gt_below[w];
      eq_below += s_eq_below[w];
    }
  } else {
    gt = eq = 0;
  }
  const uint32_t stay_below = gt_below + min(eq_below, ties);  // of the places below m
  if (tid == 0) a.moves[x.at] = m - stay_below;
  list_moves(a, x, j0, j1, held, keys, least, ties, gt, eq, stay_below);
  if (!held) x.copy(j0, j1, lane, 64);
}

// Long lines in segments, a block each: those of the first m places, then those of
// the others, so that no segment has places on both sides.  24 lines of 131001 places:
// four launches, 11, 17, 17 and 28 us; what each block adds up of the other segments'
// histograms is a third of it, so that segments of 2048 places take 45% longer in all.
struct Segment {
  int lower;   // segments below m
  int j0, j1;  // this one's places
  __device__ __forceinline__ Segment(const Line& x, int segments, int seg) {
    const int n = x.r.n, m = x.m;
    lower = min(max((int)(((int64_t)segments * m + n / 2) / n), 1), segments - 1);
    const bool low = seg < lower;
    const int base = low ? 0 : m, size = low ? m : n - m, parts = low ? lower : segments - lower, i = low ? seg : seg - lower;
    const int each = ((size + parts - 1) / parts + 63) / 64 * 64;
    j0 = __builtin_amdgcn_readfirstlane(base + (int)min((int64_t)i * each, (int64_t)size));
    j1 = __builtin_amdgcn_readfirstlane(base + (int)min((int64_t)(i + 1) * each, (int64_t)size));
  }
};
constexpr int bits_from(int round) { return round == 0 ? 21 : round == 1 ? 10 : 0; }
constexpr uint32_t bits_mask(int round) { return round == 2 ? 1023u : 2047u; }

// The bin of a round's histogram (of all segments) in which the last row that stays lies:
// its bits join those known, and of the rows that stay those among the keys with them.
template <int ROUND>
__device__ __forceinline__ uint2 find_bin(const EvictArgs& a, const Line& x) {
  __shared__ uint32_t s_wave[kSplitWaves];
  __shared__ uint2 s_found;
  constexpr int PER = kBins / kSplitThreads;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint2 known = ROUND == 0 ? make_uint2(0u, (uint32_t)x.m) : a.found[ROUND > 0 ? ROUND - 1 : 0][x.at];
  const uint4* hist = reinterpret_cast<const uint4*>(a.hist[ROUND] + x.at * a.segments * kBins);
  static_assert(PER == 4, "a thread's bins are a vector");
  const int mine = kSplitThreads - 1 - tid;  // from the top
  uint4 n = make_uint4(0, 0, 0, 0);
#pragma unroll 1
  for (int s0 = 0; s0 < a.segments; s0 += 16) {
    uint4 o[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) o[u] = hist[min(s0 + u, a.segments - 1) * (kBins / 4) + mine];
#pragma unroll
    for (int u = 0; u < 16; ++u)
      if (s0 + u < a.segments) {
        n.x += o[u].x; n.y += o[u].y; n.z += o[u].z; n.w += o[u].w;
      }
  }
  const uint32_t sum = n.x + n.y + n.z + n.w;
  uint32_t incl = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = __shfl_up(incl, off, kWave);
    if (lane >= off) incl += o;
  }
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  uint32_t before = incl - sum;
  for (int w = 0; w < wave; ++w) before += s_wave[w];
  if (before < known.y && before + sum >= known.y) {
    uint32_t bin = 4 * mine + 3, left = known.y - before;
    if (left > n.w) { left -= n.w; --bin;
      if (left > n.z) { left -= n.z; --bin;
        if (left > n.y) { left -= n.y; --bin; } } }
    s_found = make_uint2(known.x | bin << bits_from(ROUND), left);
  }
  __syncthreads();
  return s_found;
}

// A round's histogram of a segment's keys, of those that have the bits known so far.
template <int ROUND>
__global__ __launch_bounds__(kSplitThreads) void split_count_kernel(EvictArgs a) {
  __shared__ uint32_t s_keys[kSplitWaves][kWaveKeys];
  __shared__ uint32_t bins[kBins], s_larger[kSplitWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = blockIdx.x / a.segments, seg = blockIdx.x - head * a.segments;
  const Line x(a, head);
  if (x.m == x.r.n || x.m == 0) return;
  const Segment g(x, a.segments, seg);
  uint32_t known = 0;
  if constexpr (ROUND > 0) {
    const uint2 found = find_bin<ROUND - 1>(a, x);
    known = found.x;
    if (seg == 0 && tid == 0) a.found[ROUND - 1][x.at] = found;
  }
  uint32_t larger = 0;
  for (int b = tid; b < kBins; b += kSplitThreads) bins[b] = 0;
  __syncthreads();
  const int size = g.j1 - g.j0, share = ((size + kSplitWaves - 1) / kSplitWaves + 63) / 64 * 64;
  const int j0 = min(g.j0 + wave * share, g.j1), j1 = min(j0 + share, g.j1);
  sweep(x.r, j0, j1, false, s_keys[wave], [&](int, uint32_t k, bool there) {
    constexpr int above = ROUND == 0 ? 0 : bits_from(ROUND - 1);
    if (ROUND == 2) larger += __popcll(__ballot(there && k >> above > known >> above));
    if (ROUND > 0 && !__any(there && k >> above == known >> above)) return;
    if (there && (ROUND == 0 || k >> above == known >> above)) {
      const uint32_t bin = k >> bits_from(ROUND) & bits_mask(ROUND);
      // lanes with the first one's bin add at once
      const uint32_t first = __builtin_amdgcn_readfirstlane(bin);
      const uint64_t same = __ballot(bin == first);
      if (bin != first)
        atomicAdd(&bins[bin], 1u);
      else if (lane == __ffsll((unsigned long long)same) - 1)
        atomicAdd(&bins[bin], (uint32_t)__popcll(same));
    }
  });
  if (ROUND == 2 && lane == 0) s_larger[wave] = larger;
  __syncthreads();
  if (ROUND == 2 && tid == 0) {
    for (int w = 1; w < kSplitWaves; ++w) larger += s_larger[w];
    a.larger[x.at * a.segments + seg] = larger;
  }
  uint32_t* hist = a.hist[ROUND] + (x.at * a.segments + seg) * kBins;
  for (int b = tid; b < kBins; b += kSplitThreads) hist[b] = bins[b];
}

// The lists' share of a segment.  What lies above and at the last row's key in each
// segment, its histograms tell.
__global__ __launch_bounds__(kSplitThreads) void split_list_kernel(EvictArgs a) {
  __shared__ uint32_t s_keys[kSplitWaves][kWaveKeys];
  __shared__ uint32_t s_gt[kMaxSegments], s_eq[kMaxSegments], s_wgt[kSplitWaves], s_weq[kSplitWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = blockIdx.x / a.segments, seg = blockIdx.x - head * a.segments;
  const Line x(a, head);
  const int n = x.r.n, m = x.m;
  if (tid == 0 && blockIdx.x == 0 && x.layer == 0) a.stay[x.seq] = m;
  if (m == n || m == 0) {
    if (tid == 0 && seg == 0) a.moves[x.at] = 0;
    x.copy(0, m, seg * kSplitThreads + tid, a.segments * kSplitThreads);
    return;
  }
  const Segment g(x, a.segments, seg);
  const uint2 found = find_bin<2>(a, x);
  const uint32_t least = found.x, ties = found.y;
  // larger and equal keys of each segment, a wave each
  const int last = least & bits_mask(2);
  for (int s = wave; s < a.segments; s += kSplitWaves) {
    const uint4* hist = reinterpret_cast<const uint4*>(a.hist[2] + (x.at * a.segments + s) * kBins);
    uint32_t above = 0, equal = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int b = 4 * (64 * u + lane);
      const uint4 n = hist[64 * u + lane];
      above += (b > last ? n.x : 0) + (b + 1 > last ? n.y : 0) + (b + 2 > last ? n.z : 0) + (b + 3 > last ? n.w : 0);
      equal += (b == last ? n.x : 0) + (b + 1 == last ? n.y : 0) + (b + 2 == last ? n.z : 0) + (b + 3 == last ? n.w : 0);
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) {
      above += __shfl_xor(above, off, kWave);
      equal += __shfl_xor(equal, off, kWave);
    }
    if (lane == 0) {
      s_gt[s] = above + a.larger[x.at * a.segments + s];
      s_eq[s] = equal;
    }
  }
  __syncthreads();
  uint32_t gt = 0, eq = 0, gt_below = 0, eq_below = 0;
  for (int s = 0; s < a.segments; ++s) {
    if (s < seg) {
      gt += s_gt[s];
      eq += s_eq[s];
    }
    if (s < g.lower) {
      gt_below += s_gt[s];
      eq_below += s_eq[s];
    }
  }
  const uint32_t stay_below = gt_below + min(eq_below, ties);  // of the places below m
  if (tid == 0 && seg == 0) a.moves[x.at] = m - stay_below;
  // its waves' shares in turn
  const int size = g.j1 - g.j0, share = ((size + kSplitWaves - 1) / kSplitWaves + 63) / 64 * 64;
  const int j0 = min(g.j0 + wave * share, g.j1), j1 = min(j0 + share, g.j1);
  const bool held = share <= kWaveKeys;
  uint32_t* const keys = s_keys[wave];
  if (held) x.load(j0, j1, keys);
  uint32_t wgt = 0, weq = 0;
  sweep(x.r, j0, j1, held, keys, [&](int, uint32_t k, bool in) {
    wgt += __popcll(__ballot(in && k > least));
    weq += __popcll(__ballot(in && k == least));
  });
  if (lane == 0) {
    s_wgt[wave] = wgt;
    s_weq[wave] = weq;
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    gt += s_wgt[w];
    eq += s_weq[w];
  }
  list_moves(a, x, j0, j1, held, keys, least, ties, gt, eq, stay_below);
  if (!held) x.copy(j0, j1, lane, 64);
}

// Moves the rows of a line's list, 16 bytes of a key and of a value a lane at a time.
// Places that rows come from are not written, so any order will do.  Bound by memory: 8
// prompts cut to a quarter 56 us, 5.4 TB/s; 131001 rows to half in 3 layers 174 us, 4.8 TB/s.
// The stores go past the caches (the prompts 66 us with ordinary ones).
__global__ __launch_bounds__(kMoveThreads) void move_kernel(EvictArgs a, int chunks) {
  const int head = blockIdx.x / chunks, chunk = blockIdx.x - head * chunks, seq = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x;
  const int64_t line = line_of(a, layer, seq, head);
  if (tid == 0 && blockIdx.x == 0 && layer == 0) a.length_out[seq] = a.stay[seq];
  const int moves = a.moves[line];
  const int32_t *to = a.to + line * a.list_stride, *from = a.from + line * a.list_stride;
  u32x4 *k = reinterpret_cast<u32x4*>(a.c.k) + layer * a.layer16, *v = reinterpret_cast<u32x4*>(a.c.v) + layer * a.layer16;
  const int64_t head16 = head * a.c.head_stride(a.row16);
  const int per = kMoveThreads / a.row16, mine = tid / a.row16, l = tid - mine * a.row16;
  if (mine >= per) return;
  const int64_t step = (int64_t)chunks * per;
  for (int64_t i0 = (int64_t)chunk * per + mine; i0 < moves; i0 += kMoveBatch * step) {
    u32x4 x[kMoveBatch], y[kMoveBatch];
    int64_t at[kMoveBatch];
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u) {
      const int64_t i = min(i0 + u * step, (int64_t)moves - 1);
      const int dst = to[i], src = from[i];
      const int dst_page = a.c.page_of(seq, dst), src_page = a.c.page_of(seq, src);
      const bool there = dst_page >= 0 && src_page >= 0 && i0 + u * step < moves;
      at[u] = there ? a.c.row_in(dst_page, dst, a.row16) + head16 + l : -1;
      const int64_t s = a.c.row_in(max(src_page, 0), src, a.row16) + head16 + l;
      x[u] = k[s];
      y[u] = v[s];
      if (l == 0 && i0 + u * step < moves) {
        a.weights_out[line * a.stride + dst] = a.weights[line * a.stride + src];
        if (a.born) a.born_out[line * a.stride + dst] = a.born[line * a.stride + src];
      }
    }
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u)
      if (at[u] >= 0) {
        __builtin_nontemporal_store(x[u], k + at[u]);
        __builtin_nontemporal_store(y[u], v + at[u]);
      }
  }
}

uint64_t align16(uint64_t n) { return (n + 15) / 16 * 16; }

// Moves of a line, at most: as many places free as rows that move.
uint64_t most_moves(const mit2cfm_kv_cache& c, const mit2cfm_kv_evict& p) {
  return std::min<uint64_t>(p.weight_stride, (uint64_t)c.table_stride * c.page_rows) / 2 + 1;
}
// Segments of a line, an eighth shorter than a block's waves hold; 1: one block's registers
// hold the line.  (256 lines of 16000 places 216 us in a block each, 241 in segments, 32 of
// them 62 and 54; of 20000 places 327 and 291, 136 and 61.)
int segments_of(const mit2cfm_kv_cache& c, const mit2cfm_kv_evict& p) {
  const uint64_t len = std::min<uint64_t>({p.max_length, p.weight_stride, (uint64_t)c.table_stride * c.page_rows});
  const uint64_t lines = (uint64_t)p.layers * p.seqs * c.kv_heads;
  if (len <= 16 * kWaveKeys) return 1;
  // (with room: what lies below the budget is divided by itself)
  return (int)std::min<uint64_t>({len / (kSplitKeys * 7 / 8) + 1, (uint64_t)kMaxSegments, std::max<uint64_t>(2, 4096 / lines)});
}
bool evict_in_range(const mit2cfm_kv_cache& c, const mit2cfm_kv_evict& p) {
  return p.seqs <= 65535 && p.layers >= 1 && p.layers <= 16384 && (uint64_t)p.layers * p.seqs * c.kv_heads <= (1u << 24) &&
         p.weight_stride >= 1 && p.weight_stride <= (1u << 30);
}

}  // namespace

uint64_t kv_evict_workspace(const mit2cfm_kv_cache& c, const mit2cfm_kv_evict& p) {
  try {
    check_kv_sizes(c);
  } catch (const std::invalid_argument&) {
    return 0;
  }
  if (p.seqs == 0 || !evict_in_range(c, p)) return 0;
  const uint64_t lines = (uint64_t)p.layers * p.seqs * c.kv_heads;
  const uint64_t segments = (uint64_t)segments_of(c, p);
  return 2 * align16(lines * most_moves(c, p) * 4) + align16(lines * 4) + align16(p.seqs * 4) +
         (segments > 1 ? 3 * lines * segments * kBins * 4 + 2 * align16(lines * 8) + align16(lines * segments * 4) : 0);
}

void kv_evict(const mit2cfm_kv_cache& c, const mit2cfm_kv_evict& p, hipStream_t s) {
  check_kv_cache(c);
  need(evict_in_range(c, p),
       "seqs must be <= 65535, layers in [1, 16384], layers * seqs * kv_heads <= 2^24, weight_stride in [1, 2^30]");
  need(p.layers == 1 || p.layer_stride % 8 == 0, "layer_stride must be a multiple of 8");
  need(p.layers == 1 || p.layer_stride >= (uint64_t)c.pages * c.kv_heads * c.page_rows * c.head_dim,
       "layer_stride is smaller than a layer");
  if (p.seqs == 0) return;
  need(p.length && p.keep && p.weights && p.weights_out && p.length_out,
       "length, keep, weights, weights_out and length_out must not be NULL");
  need(!p.born == !p.born_out && !p.born == !p.now, "born, born_out and now belong together");
  need(aligned(p.length, 4) && aligned(p.keep, 4) && aligned(p.weights, 4) && aligned(p.weights_out, 4) && aligned(p.born, 4) &&
           aligned(p.born_out, 4) && aligned(p.now, 4) && aligned(p.length_out, 4),
       "length, keep, weights, born, now and the outputs must be 4-byte aligned");
  const uint64_t lines = (uint64_t)p.layers * p.seqs * c.kv_heads, bytes = lines * p.weight_stride * 4, seq_bytes = p.seqs * 4ull;
  need(p.weights == p.weights_out || !meet(p.weights, bytes, p.weights_out, bytes), "weights_out overlaps weights");
  if (p.born) {
    need(p.born == p.born_out || !meet(p.born, bytes, p.born_out, bytes), "born_out overlaps born");
    need(!meet(p.weights, bytes, p.born_out, bytes) && !meet(p.weights_out, bytes, p.born, bytes) &&
             !meet(p.weights_out, bytes, p.born_out, bytes) && !meet(p.now, seq_bytes, p.weights_out, bytes) &&
             !meet(p.now, seq_bytes, p.born_out, bytes) && !meet(p.now, seq_bytes, p.length_out, seq_bytes),
         "weights, born, now and their outputs overlap");
  }
  auto clear = [&](const void* out, uint64_t n) {
    const bool length = out == p.length_out && p.length == p.length_out;  // (may be itself)
    return !meet(p.keep, seq_bytes, out, n) && (length || !meet(p.length, seq_bytes, out, n));
  };
  need(clear(p.weights_out, bytes) && clear(p.length_out, seq_bytes) && (!p.born || clear(p.born_out, bytes)) &&
           !meet(p.weights, bytes, p.length_out, seq_bytes) && !meet(p.weights_out, bytes, p.length_out, seq_bytes) &&
           !(p.born && (meet(p.born, bytes, p.length_out, seq_bytes) || meet(p.born_out, bytes, p.length_out, seq_bytes))),
       "an output overlaps length, keep or another buffer");
  need(p.workspace && p.workspace_bytes >= kv_evict_workspace(c, p), "workspace is NULL or too small");
  need(aligned(p.workspace, 16), "workspace must be 16-byte aligned");
  EvictArgs a{};
  a.c = view(c);
  a.length = p.length; a.keep = p.keep;
  a.weights = p.weights; a.weights_out = p.weights_out;
  a.born = p.born; a.born_out = p.born_out; a.now = p.now;
  a.length_out = p.length_out;
  a.stride = p.weight_stride;
  const int e = kv_elem_bytes(c.dtype);
  a.layer16 = p.layers > 1 ? (int64_t)(p.layer_stride * e / 16) : 0;
  a.row16 = (int)c.head_dim * e / 16;
  a.seqs = (int)p.seqs;
  a.first_rows = p.first_rows;
  a.last_rows = p.last_rows;
  a.list_stride = (int64_t)most_moves(c, p);
  char* w = static_cast<char*>(p.workspace);
  a.to = reinterpret_cast<int32_t*>(w);
  w += align16(lines * a.list_stride * 4);
  a.from = reinterpret_cast<int32_t*>(w);
  w += align16(lines * a.list_stride * 4);
  a.moves = reinterpret_cast<int32_t*>(w);
  w += align16(lines * 4);
  a.stay = reinterpret_cast<int32_t*>(w);
  w += align16(p.seqs * 4);
  const uint64_t len = std::min<uint64_t>({p.max_length, p.weight_stride, (uint64_t)c.table_stride * c.page_rows});
  a.segments = segments_of(c, p);
  const dim3 grid(c.kv_heads * a.segments, p.seqs, p.layers);
  if (a.segments > 1) {
    for (int round = 0; round < 3; ++round) {
      a.hist[round] = reinterpret_cast<uint32_t*>(w);
      w += lines * a.segments * kBins * 4;
    }
    for (int round = 0; round < 2; ++round) {
      a.found[round] = reinterpret_cast<uint2*>(w);
      w += align16(lines * 8);
    }
    a.larger = reinterpret_cast<uint32_t*>(w);
    hipLaunchKernelGGL((split_count_kernel<0>), grid, dim3(kSplitThreads), 0, s, a);
    kv_launched(hipGetLastError());
    hipLaunchKernelGGL((split_count_kernel<1>), grid, dim3(kSplitThreads), 0, s, a);
    kv_launched(hipGetLastError());
    hipLaunchKernelGGL((split_count_kernel<2>), grid, dim3(kSplitThreads), 0, s, a);
    kv_launched(hipGetLastError());
    hipLaunchKernelGGL(split_list_kernel, grid, dim3(kSplitThreads), 0, s, a);
  } else if (len <= kWaveKeys) {
    hipLaunchKernelGGL((choose_kernel<1>), grid, dim3(64), 0, s, a);
  } else if (len <= 4 * kWaveKeys) {
    hipLaunchKernelGGL((choose_kernel<4>), grid, dim3(256), 0, s, a);
  } else if (len <= 8 * kWaveKeys) {
    hipLaunchKernelGGL((choose_kernel<8>), grid, dim3(512), 0, s, a);
  } else {
    hipLaunchKernelGGL((choose_kernel<16>), grid, dim3(1024), 0, s, a);
  }
  kv_launched(hipGetLastError());
  // 16 blocks a CU, of a line no more than its moves want, half its places at most: 256
  // lines of 2048 moves 75 us (4 a CU 80); but lines that are 4 a CU themselves have one
  // block each: 1440 of them with a move each 10.7 us (two blocks each 11.9, eleven 17.2).
  const uint64_t per = kMoveThreads / a.row16 * kMoveBatch;
  const uint64_t wanted = lines >= 1024 ? 1 : 4096 / lines;
  const int chunks = (int)std::min(wanted, (len / 2 + per - 1) / per + 1);
  hipLaunchKernelGGL(move_kernel, dim3(c.kv_heads * chunks, p.seqs, p.layers), dim3(kMoveThreads), 0, s, a, chunks);
  kv_launched(hipGetLastError());
}

}  // namespace mit2hip
