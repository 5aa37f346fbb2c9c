// kv_evict.hip -- rows of least weight leave a paged cache (see kv_ops.h and
// mit2cfm.h for what it computes).
#include <algorithm>

#include "kv_args.h"

namespace mit2hip {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kChooseThreads = 1024, kChooseWaves = kChooseThreads / 64;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;

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
  int64_t oldest;                         // with births: rows from this one on
  __device__ __forceinline__ uint32_t key(int j) const {
    const bool stays = j < first || (born ? (int64_t)born[j] >= oldest : j >= tail);
    uint32_t u = __float_as_uint(weights[j]);
    if (u == 0x80000000u) u = 0;
    const bool least = (u & 0x7fffffffu) > 0x7f800000u || (unsigned)table[j >> page_shift] >= (unsigned)pages;
    u ^= u >> 31 ? 0xffffffffu : 0x80000000u;
    return stays ? 0xffffffffu : least ? 0u : u;
  }
};

// A block ranks a line: the key of the last row that stays is found by three
// histograms of its bits (11, 11, 10), among the keys that agree so far; then each
// wave walks its share of the places in order.  A place p that stays has
// before(p) = #(larger keys before p) + min(#(equal keys before p), ties) rows before
// it that stay, which gives a freed place and a row that moves their numbers in the
// lists: p - before(p), before(p) - before(keep).
__global__ __launch_bounds__(kChooseThreads) void choose_kernel(EvictArgs a) {
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t s_wave[kChooseWaves], s_gt[kChooseWaves], s_eq[kChooseWaves], s_gt_below[kChooseWaves], s_eq_below[kChooseWaves];
  __shared__ uint32_t s_bin, s_left;
  const int head = blockIdx.x, seq = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const int64_t line = line_of(a, layer, seq, head);
  Ranks r;
  r.n = places_of(a, seq);
  const int m = min(r.n, max(a.keep[seq], 0));
  const bool apart = a.weights_out != a.weights, apart_born = a.born && a.born_out != a.born;
  r.weights = a.weights + line * a.stride;
  r.born = a.born ? a.born + line * a.stride : nullptr;
  r.table = a.c.table + (size_t)seq * a.c.table_stride;
  r.first = (int)min(a.first_rows, (int64_t)r.n);
  r.tail = (int)max(r.n - a.last_rows, (int64_t)0);
  r.pages = a.c.pages;
  r.page_shift = a.c.page_shift;
  r.oldest = a.born ? (int64_t)a.now[seq] - a.last_rows : 0;
  float* weights_out = a.weights_out + line * a.stride;
  int32_t* born_out = a.born_out ? a.born_out + line * a.stride : nullptr;
  if (tid == 0 && head == 0 && layer == 0) a.stay[seq] = m;
  if (m == r.n || m == 0) {
    if (tid == 0) a.moves[line] = 0;
    for (int j = tid; j < m; j += blockDim.x) {
      if (apart) weights_out[j] = r.weights[j];
      if (apart_born) born_out[j] = r.born[j];
    }
    return;
  }

  uint32_t agreed = 0, left = m;  // the bits so far; rows that stay among the keys that have them
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, above = round == 0 ? 32 : round == 1 ? 21 : 10;
    const uint32_t mask = round == 2 ? 1023u : 2047u;
    for (int b = tid; b < kBins; b += blockDim.x) bins[b] = 0;
    __syncthreads();
    for (int j = tid; j < r.n; j += blockDim.x) {
      const uint32_t k = r.key(j);
      const bool in = round == 0 || k >> above == agreed >> above;
      if (!in) continue;
      const uint32_t bin = k >> shift & mask;
      // lanes with the first one's bin add at once
      const uint32_t first = __builtin_amdgcn_readfirstlane(bin);
      const uint64_t same = __ballot(bin == first);
      if (bin != first)
        atomicAdd(&bins[bin], 1u);
      else if (lane == __ffsll((unsigned long long)same) - 1)
        atomicAdd(&bins[bin], (uint32_t)__popcll(same));
    }
    __syncthreads();
    // from the top: the bin in which the last row that stays lies
    const int per = kBins / blockDim.x;  // a thread's bins, neighbours
    const int top = kBins - 1 - tid * per;
    uint32_t mine = 0;
    for (int b = 0; b < per; ++b) mine += bins[top - b];
    uint32_t incl = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t o = __shfl_up(incl, off, kWave);
      if (lane >= off) incl += o;
    }
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    uint32_t before = incl - mine;
    for (int w = 0; w < wave; ++w) before += s_wave[w];
    if (before < left && before + mine >= left) {
      for (int b = 0; b < per; ++b) {
        const uint32_t n = bins[top - b];
        if (before + n >= left) {
          s_bin = top - b;
          s_left = left - before;
          break;
        }
        before += n;
      }
    }
    __syncthreads();
    agreed |= s_bin << shift;
    left = s_left;
    __syncthreads();
  }
  const uint32_t least = agreed, ties = left;  // keys above `least` stay, and the first `ties` that equal it

  // each wave's places, a multiple of 64
  const int share = ((r.n + waves - 1) / waves + 63) / 64 * 64;
  const int j0 = min(wave * share, r.n), j1 = min(j0 + share, r.n);
  uint32_t gt = 0, eq = 0, gt_below = 0, eq_below = 0;
  for (int j = j0 + lane; j < j1; j += 64) {
    const uint32_t k = r.key(j);
    gt += k > least;
    eq += k == least;
    gt_below += k > least && j < m;
    eq_below += k == least && j < m;
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    gt += __shfl_xor(gt, off, kWave);
    eq += __shfl_xor(eq, off, kWave);
    gt_below += __shfl_xor(gt_below, off, kWave);
    eq_below += __shfl_xor(eq_below, off, kWave);
  }
  if (lane == 0) {
    s_gt[wave] = gt;
    s_eq[wave] = eq;
    s_gt_below[wave] = gt_below;
    s_eq_below[wave] = eq_below;
  }
  __syncthreads();
  gt = eq = gt_below = eq_below = 0;
  for (int w = 0; w < waves; ++w) {
    if (w < wave) {
      gt += s_gt[w];
      eq += s_eq[w];
    }
    gt_below += s_gt_below[w];
    eq_below += s_eq_below[w];
  }
  const uint32_t stay_below = gt_below + min(eq_below, ties);  // of the places below m
  if (tid == 0) a.moves[line] = m - stay_below;
  int32_t *to = a.to + line * a.list_stride, *from = a.from + line * a.list_stride;
  for (int j = j0 + lane; j - lane < j1; j += 64) {
    const bool in = j < j1;
    const uint32_t k = in ? r.key(j) : 0;
    const bool more = in && k > least, equal = in && k == least;
    const uint64_t below = (1ull << lane) - 1, vote_gt = __ballot(more), vote_eq = __ballot(equal);
    const uint32_t gt_before = gt + __popcll(vote_gt & below), eq_before = eq + __popcll(vote_eq & below);
    const uint32_t before = gt_before + min(eq_before, ties);
    const bool stays = more || (equal && eq_before < ties);
    if (in && j < m) {
      if (!stays) {
        to[j - before] = j;
      } else {
        if (apart) weights_out[j] = r.weights[j];
        if (apart_born) born_out[j] = r.born[j];
      }
    } else if (stays) {
      from[before - stay_below] = j;
    }
    gt += __popcll(vote_gt);
    eq += __popcll(vote_eq);
  }
}

// Moves the rows of a line's list, 16 bytes of a key and of a value a lane at a time.
// Places that rows come from are not written, so any order will do.
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
  for (int64_t i = (int64_t)chunk * per + mine; i < moves; i += (int64_t)chunks * per) {
    const int dst = to[i], src = from[i];
    const int dst_page = a.c.page_of(seq, dst), src_page = a.c.page_of(seq, src);
    if (l == 0) {
      a.weights_out[line * a.stride + dst] = a.weights[line * a.stride + src];
      if (a.born) a.born_out[line * a.stride + dst] = a.born[line * a.stride + src];
    }
    if (dst_page < 0 || src_page < 0) continue;
    const int64_t d = a.c.row_in(dst_page, dst, a.row16) + head16 + l, s = a.c.row_in(src_page, src, a.row16) + head16 + l;
    k[d] = k[s];
    v[d] = v[s];
  }
}

uint64_t align16(uint64_t n) { return (n + 15) / 16 * 16; }

// Moves of a line, at most: as many places free as rows that move.
uint64_t most_moves(const mit2cfm_kv_cache& c, const mit2cfm_kv_evict& p) {
  return std::min<uint64_t>(p.weight_stride, (uint64_t)c.table_stride * c.page_rows) / 2 + 1;
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
  return 2 * align16(lines * most_moves(c, p) * 4) + align16(lines * 4) + align16(p.seqs * 4);
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
  const uint64_t len = std::min<uint64_t>({p.max_length, p.weight_stride, (uint64_t)c.table_stride * c.page_rows});
  // as many threads as a thread has about eight places each
  const int threads = len <= 2048 ? 256 : len <= 4096 ? 512 : kChooseThreads;
  hipLaunchKernelGGL(choose_kernel, dim3(c.kv_heads, p.seqs, p.layers), dim3(threads), 0, s, a);
  kv_launched(hipGetLastError());
  const uint64_t per = kMoveThreads / a.row16;
  const uint64_t wanted = std::max<uint64_t>(1, 8192 / lines);  // blocks of a line, for as many moves as half its places at most
  const int chunks = (int)std::min(wanted, (len / 2 + per - 1) / per + 1);
  hipLaunchKernelGGL(move_kernel, dim3(c.kv_heads * chunks, p.seqs, p.layers), dim3(kMoveThreads), 0, s, a, chunks);
  kv_launched(hipGetLastError());
}

}  // namespace mit2hip
