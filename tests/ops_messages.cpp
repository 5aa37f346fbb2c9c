// Calls the cache and beam operators with arguments that are sound but for one, and
// looks for that one in the message of the refusal.  Every call is refused before a
// GPU is touched.  Exit status 1 when one was not, or for another reason.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <stdexcept>

#include "mit2cfm.h"

typedef struct ihipStream_t* hipStream_t;
namespace mit2hip {
void kv_append(const mit2cfm_kv_cache&, const mit2cfm_kv_rows&, const mit2cfm_kv_append&, hipStream_t);
void kv_attention(const mit2cfm_kv_cache&, const mit2cfm_kv_rows&, const mit2cfm_kv_attention&, hipStream_t);
void beam_select(const mit2cfm_beam_select&, hipStream_t);
void beam_reorder(const mit2cfm_kv_cache&, const mit2cfm_beam_reorder&, hipStream_t);
}  // namespace mit2hip

// buffers of their own: 4 KB apart
alignas(4096) static char mem[24][4096];
static int bad = 0, tried = 0;

static void refused(const char* what, const char* why, const std::function<void()>& call) {
  ++tried;
  try {
    call();
  } catch (const std::invalid_argument& e) {
    if (std::strstr(e.what(), why)) return;
    std::printf("%s: refused for \"%s\", not for \"%s\"\n", what, e.what(), why);
    ++bad;
    return;
  } catch (const std::exception& e) {
    std::printf("not refused as an argument: %s (%s)\n", what, e.what());
    ++bad;
    return;
  }
  std::printf("not refused: %s\n", what);
  ++bad;
}
template <typename T>
static T* at(int n, size_t off = 0) {
  return reinterpret_cast<T*>(mem[n] + off);
}

static mit2cfm_kv_cache cache() {
  mit2cfm_kv_cache c{};
  c.k = mem[20]; c.v = mem[21];
  c.table = at<int32_t>(0);
  c.pages = 2; c.page_rows = 2; c.kv_heads = 2; c.head_dim = 64; c.table_stride = 2;
  c.dtype = MIT2CFM_DTYPE_F16;
  return c;
}
static mit2cfm_kv_rows rows() {
  mit2cfm_kv_rows r{};
  r.start = at<int32_t>(1); r.length = at<int32_t>(2);
  r.seqs = 1; r.rows = 2; r.max_length = 3;
  return r;
}
static mit2cfm_kv_append append() {  // (2 rows of 4 heads of 64 f16: 1 KB)
  mit2cfm_kv_append a{};
  a.k = mem[3]; a.v = mem[4]; a.q = mem[5]; a.q_out = mem[6];
  a.k_row = a.v_row = 128; a.k_head = a.v_head = a.q_head = a.q_out_head = 64;
  a.q_row = a.q_out_row = 256; a.q_heads = 4;
  a.rotary_dim = 64; a.theta = 10000.0;
  return a;
}
static mit2cfm_kv_attention attention() {
  mit2cfm_kv_attention a{};
  a.q = mem[5]; a.out = mem[6];
  a.q_row = a.out_row = 256; a.q_head = a.out_head = 64; a.q_heads = 4; a.scale = 0.125f;
  a.workspace = mem[7]; a.workspace_bytes = ~0ull;
  return a;
}
static mit2cfm_beam_select select_args() {
  mit2cfm_beam_select a{};
  a.logits = mem[8]; a.logits_row = 100; a.groups = 3; a.beams = 2; a.vocab = 100; a.count = 4;
  a.scores = at<float>(9); a.finished = at<int32_t>(10); a.stop_token = 7;
  a.scores_out = at<float>(11); a.parent_out = at<int32_t>(12); a.token_out = at<int32_t>(13); a.finished_out = at<int32_t>(14);
  a.workspace = mem[15]; a.workspace_bytes = ~0ull;
  return a;
}
static mit2cfm_beam_reorder reorder_args() {
  mit2cfm_beam_reorder a{};
  a.groups = 1; a.beams = 2; a.layers = 2; a.layer_stride = 2 * 2 * 2 * 64;
  a.parent = at<int32_t>(9); a.length = at<int32_t>(10); a.parent_stride = 2;
  a.table_out = at<int32_t>(11);
  a.state = at<uint32_t>(12); a.state_out = at<uint32_t>(13); a.state_words = 3;
  a.token = at<uint32_t>(14); a.place = at<int32_t>(15);
  return a;
}

#define CACHE(why, ...) { auto c = cache(); c.__VA_ARGS__; \
    refused("append: cache " #__VA_ARGS__, why, [&] { mit2hip::kv_append(c, rows(), append(), nullptr); }); \
    refused("attention: cache " #__VA_ARGS__, why, [&] { mit2hip::kv_attention(c, rows(), attention(), nullptr); }); \
    refused("reorder: cache " #__VA_ARGS__, why, [&] { mit2hip::beam_reorder(c, reorder_args(), nullptr); }); }
#define ROWS(why, ...) { auto r = rows(); r.__VA_ARGS__; \
    refused("append: rows " #__VA_ARGS__, why, [&] { mit2hip::kv_append(cache(), r, append(), nullptr); }); \
    refused("attention: rows " #__VA_ARGS__, why, [&] { mit2hip::kv_attention(cache(), r, attention(), nullptr); }); }
#define APPEND(why, ...) { auto a = append(); a.__VA_ARGS__; \
    refused("append: " #__VA_ARGS__, why, [&] { mit2hip::kv_append(cache(), rows(), a, nullptr); }); }
#define ATTEND(why, ...) { auto a = attention(); a.__VA_ARGS__; \
    refused("attention: " #__VA_ARGS__, why, [&] { mit2hip::kv_attention(cache(), rows(), a, nullptr); }); }
#define SELECT(why, ...) { auto a = select_args(); a.__VA_ARGS__; \
    refused("select: " #__VA_ARGS__, why, [&] { mit2hip::beam_select(a, nullptr); }); }
#define REORDER(why, ...) { auto a = reorder_args(); a.__VA_ARGS__; \
    refused("reorder: " #__VA_ARGS__, why, [&] { mit2hip::beam_reorder(cache(), a, nullptr); }); }

int main() {
  // buffers that lie on one another, wholly or in part
  APPEND("q_out's rows and heads", q_out_row = 64) APPEND("q_out's rows and heads", q_out_row = 128, a.q_out_head = 128)
  APPEND("q_out's rows and heads", q_out_head = 96, a.q_out_row = 300) APPEND("q_out's rows and heads", q_out_row = 255)
  APPEND("only with its strides", q_out = mem[5], a.q_out_row = 512)
  APPEND("q_out overlaps q", q_out = mem[5] + 128) APPEND("q_out overlaps q", q_out = mem[5] - 1022) APPEND("q_out overlaps q", q_out = mem[5] + 512)
  APPEND("q_out overlaps q", q_out = mem[5] + 1022) APPEND("q_out overlaps q", q_out = mem[5] + 128, a.q_row = 0)
  APPEND("q_out overlaps k or v", q_out = mem[3]) APPEND("q_out overlaps k or v", q_out = mem[4] + 510)
  APPEND("q_out overlaps k or v", v = mem[5] + 448, a.v_row = 256, a.q_out = mem[5])  // (a head early in a packed row)
  ATTEND("out's rows and heads", out_row = 64) ATTEND("out's rows and heads", out_row = 128, a.out_head = 128)
  ATTEND("nor the same", out = mem[5]) ATTEND("out overlaps q", out = mem[5] + 512) ATTEND("out overlaps q", out = mem[5] - 512)
  ATTEND("out overlaps q", out = mem[5] + 128, a.out_row = 64, a.out_head = 128)
  SELECT("scores_out must not", scores_out = at<float>(9)) SELECT("scores_out must not", scores_out = at<float>(9, 20))
  SELECT("scores_out must not", scores = at<float>(11, 44))
  SELECT("finished_out finished", finished_out = at<int32_t>(10)) SELECT("finished_out finished", finished_out = at<int32_t>(10, 20))
  REORDER("table_out overlaps", table_out = at<int32_t>(0)) REORDER("table_out overlaps", table_out = at<int32_t>(0, 12))
  REORDER("state_out overlaps", state_out = at<uint32_t>(12)) REORDER("state_out overlaps", state = at<uint32_t>(13, 20))
  REORDER("smaller than a layer", layer_stride = 504) REORDER("smaller than a layer", layer_stride = 8) REORDER("smaller than a layer", layer_stride = 0)

  // each other argument by itself
  CACHE("must not be NULL", k = nullptr) CACHE("must not be NULL", v = nullptr) CACHE("must not be NULL", table = nullptr)
  CACHE("16-byte aligned", k = mem[20] + 8) CACHE("16-byte aligned", v = mem[20] + 4) CACHE("4-byte aligned", table = at<int32_t>(0, 2))
  CACHE("pages must", pages = 0) CACHE("pages must", pages = 1u << 31) CACHE("page_rows must", page_rows = 0) CACHE("page_rows must", page_rows = 24)
  CACHE("page_rows must", page_rows = 2048) CACHE("kv_heads must", kv_heads = 0) CACHE("kv_heads must", kv_heads = 1025)
  CACHE("head_dim must", head_dim = 0) CACHE("head_dim must", head_dim = 48) CACHE("head_dim must", head_dim = 512)
  CACHE("table_stride must", table_stride = 0) CACHE("table_stride must", table_stride = (1u << 29) + 1)
  CACHE("dtype must", dtype = 3) CACHE("dtype must", dtype = -1)
  ROWS("start and length must not", start = nullptr) ROWS("start and length must not", length = nullptr) ROWS("seqs must", seqs = 65536)
  ROWS("rows must be below", rows = 1u << 24) ROWS("4-byte aligned", start = at<int32_t>(1, 1)) ROWS("4-byte aligned", length = at<int32_t>(1, 2))
  APPEND("k and v must not", k = nullptr) APPEND("k and v must not", v = nullptr) APPEND("aligned to their type", k = mem[3] + 1)
  APPEND("aligned to their type", v = mem[4] + 3) APPEND("aligned to their type", q = mem[5] + 1) APPEND("aligned to their type", q_out = mem[6] + 1)
  APPEND("q needs q_out", q_out = nullptr) APPEND("q needs q_out", q_heads = 0) APPEND("q_heads must", q_heads = 4097)
  APPEND("rotary_dim must", rotary_dim = 3) APPEND("rotary_dim must", rotary_dim = 66)
  APPEND("theta must", theta = 0.0) APPEND("theta must", theta = -1.0) APPEND("theta must", theta = NAN) APPEND("theta must", theta = INFINITY)
  APPEND("position must", position = at<int32_t>(7, 2))
  ATTEND("must not be NULL", q = nullptr) ATTEND("must not be NULL", out = nullptr) ATTEND("aligned to their type", q = mem[5] + 1)
  ATTEND("aligned to their type", out = mem[6] + 1) ATTEND("q_heads must", q_heads = 0) ATTEND("q_heads must", q_heads = 3)
  ATTEND("q_heads must", q_heads = 4098) ATTEND("scale must", scale = NAN) ATTEND("scale must", scale = INFINITY)
  ATTEND("mask_words must", mask = at<uint32_t>(16)) ATTEND("mask_words must", mask = at<uint32_t>(16), a.mask_words = 1u << 24)
  ATTEND("mask must be", mask = at<uint32_t>(16, 2), a.mask_words = 1) ATTEND("workspace must be", workspace = mem[7] + 8)
  SELECT("must not be NULL", logits = nullptr) SELECT("must not be NULL", scores = nullptr) SELECT("must not be NULL", scores_out = nullptr)
  SELECT("must not be NULL", parent_out = nullptr) SELECT("must not be NULL", token_out = nullptr) SELECT("logits must be", logits = mem[8] + 2)
  SELECT("out of range", dtype = 3) SELECT("out of range", dtype = -1) SELECT("out of range", beams = 0) SELECT("out of range", beams = 65)
  SELECT("out of range", vocab = 0) SELECT("out of range", vocab = (1u << 24) + 1) SELECT("out of range", count = 0) SELECT("out of range", count = 65)
  SELECT("out of range", count = 3, a.beams = 1, a.vocab = 2) SELECT("out of range", groups = (1u << 19) + 1)
  SELECT("stop_token must", stop_token = 100) SELECT("stop_token must", stop_token = -2) SELECT("finished needs", stop_token = -1)
  SELECT("4-byte aligned", scores = at<float>(9, 2)) SELECT("4-byte aligned", parent_out = at<int32_t>(12, 1))
  SELECT("4-byte aligned", finished_out = at<int32_t>(14, 3)) SELECT("workspace is NULL", workspace = nullptr)
  SELECT("workspace is NULL", workspace_bytes = 15) SELECT("workspace must be", workspace = mem[15] + 8)
  REORDER("beams must", beams = 0) REORDER("beams must", beams = 65) REORDER("groups * beams", groups = (1u << 19) + 1) REORDER("layers must", layers = 0)
  REORDER("layers must", layers = 16385) REORDER("multiple of 8", layer_stride = 516) REORDER("parent_stride must", parent_stride = 1)
  REORDER("must not be NULL", parent = nullptr) REORDER("must not be NULL", length = nullptr) REORDER("must not be NULL", table_out = nullptr)
  REORDER("state needs", state_out = nullptr) REORDER("state needs", state_words = 0) REORDER("state needs", state_words = 1u << 31)
  REORDER("token needs", state = nullptr) REORDER("token needs", place = nullptr) REORDER("4-byte aligned", parent = at<int32_t>(9, 2))
  REORDER("4-byte aligned", state = at<uint32_t>(12, 1)) REORDER("4-byte aligned", place = at<int32_t>(15, 2))
  std::printf("%d tried, %d wrong\n", tried, bad);
  return bad ? 1 : 0;
}
