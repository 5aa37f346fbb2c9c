// Calls the operators for long and shared contexts with arguments that are sound but for
// one, and looks for that one in the message of the refusal; prints the sizes and last
// offsets of their structures.  Every call is refused before a GPU is touched.  Exit
// status 1 when one was not, or for another reason.
#include <cmath>
#include <cstddef>
#include <cstdio>
#include <cstring>
#include <functional>
#include <stdexcept>

#include "mit2cfm.h"

typedef struct ihipStream_t* hipStream_t;
namespace mit2hip {
void kv_norm_append(const mit2cfm_kv_cache&, const mit2cfm_kv_rows&, const mit2cfm_kv_append&, const mit2cfm_kv_norm&, hipStream_t);
void kv_prefix_attention(const mit2cfm_kv_cache&, const mit2cfm_kv_rows&, const mit2cfm_kv_attention&, const mit2cfm_kv_prefix&, hipStream_t);
void kv_weigh(const mit2cfm_kv_cache&, const mit2cfm_kv_rows&, const mit2cfm_kv_weigh&, hipStream_t);
void kv_evict(const mit2cfm_kv_cache&, const mit2cfm_kv_evict&, hipStream_t);
}  // namespace mit2hip

// buffers of their own: 4 KB apart
alignas(4096) static char mem[32][4096];
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
static mit2cfm_kv_norm norm() {
  mit2cfm_kv_norm n{};
  n.q_weight = mem[7]; n.k_weight = mem[8];
  n.weight_dtype = MIT2CFM_DTYPE_F16; n.eps = 1e-6f;
  return n;
}
static mit2cfm_kv_attention attention() {
  mit2cfm_kv_attention a{};
  a.q = mem[5]; a.out = mem[6];
  a.q_row = a.out_row = 256; a.q_head = a.out_head = 64; a.q_heads = 4; a.scale = 0.125f;
  a.workspace = mem[9]; a.workspace_bytes = ~0ull;
  return a;
}
static mit2cfm_kv_prefix prefix() {
  mit2cfm_kv_prefix x{};
  x.group = at<int32_t>(10); x.shared = at<int32_t>(11); x.groups = 1; x.max_shared = 2; x.lse = at<float>(12);
  return x;
}
static mit2cfm_kv_weigh weigh() {
  mit2cfm_kv_weigh w{};
  w.q = mem[5]; w.q_row = 256; w.q_head = 64; w.q_heads = 4; w.scale = 0.125f;
  w.lse = at<float>(12); w.weights = at<float>(13); w.weights_out = at<float>(14); w.weight_stride = 4; w.decay = 1.0f;
  w.position = at<int32_t>(15); w.born = at<int32_t>(16);
  return w;
}
static mit2cfm_kv_evict evict() {
  mit2cfm_kv_evict e{};
  e.seqs = 2; e.layers = 2; e.layer_stride = 2 * 2 * 2 * 64;
  e.length = at<int32_t>(2); e.keep = at<int32_t>(17); e.max_length = 4;
  e.weights = at<float>(13); e.weights_out = at<float>(14); e.weight_stride = 4;
  e.born = at<int32_t>(15); e.born_out = at<int32_t>(16); e.now = at<int32_t>(18); e.length_out = at<int32_t>(19);
  e.workspace = mem[9]; e.workspace_bytes = ~0ull;
  return e;
}

#define CACHE(why, ...) { auto c = cache(); c.__VA_ARGS__; \
    refused("norm: cache " #__VA_ARGS__, why, [&] { mit2hip::kv_norm_append(c, rows(), append(), norm(), nullptr); }); \
    refused("prefix: cache " #__VA_ARGS__, why, [&] { mit2hip::kv_prefix_attention(c, rows(), attention(), prefix(), nullptr); }); \
    refused("weigh: cache " #__VA_ARGS__, why, [&] { mit2hip::kv_weigh(c, rows(), weigh(), nullptr); }); \
    refused("evict: cache " #__VA_ARGS__, why, [&] { mit2hip::kv_evict(c, evict(), nullptr); }); }
#define ROWS(why, ...) { auto r = rows(); r.__VA_ARGS__; \
    refused("norm: rows " #__VA_ARGS__, why, [&] { mit2hip::kv_norm_append(cache(), r, append(), norm(), nullptr); }); \
    refused("prefix: rows " #__VA_ARGS__, why, [&] { mit2hip::kv_prefix_attention(cache(), r, attention(), prefix(), nullptr); }); \
    refused("weigh: rows " #__VA_ARGS__, why, [&] { mit2hip::kv_weigh(cache(), r, weigh(), nullptr); }); }
#define APPEND(why, ...) { auto a = append(); a.__VA_ARGS__; \
    refused("norm: append " #__VA_ARGS__, why, [&] { mit2hip::kv_norm_append(cache(), rows(), a, norm(), nullptr); }); }
#define NORM(why, ...) { auto n = norm(); n.__VA_ARGS__; \
    refused("norm: " #__VA_ARGS__, why, [&] { mit2hip::kv_norm_append(cache(), rows(), append(), n, nullptr); }); }
#define ATTEND(why, ...) { auto a = attention(); a.__VA_ARGS__; \
    refused("prefix: attention " #__VA_ARGS__, why, [&] { mit2hip::kv_prefix_attention(cache(), rows(), a, prefix(), nullptr); }); }
#define PREFIX(why, ...) { auto x = prefix(); x.__VA_ARGS__; \
    refused("prefix: " #__VA_ARGS__, why, [&] { mit2hip::kv_prefix_attention(cache(), rows(), attention(), x, nullptr); }); }
#define WEIGH(why, ...) { auto w = weigh(); w.__VA_ARGS__; \
    refused("weigh: " #__VA_ARGS__, why, [&] { mit2hip::kv_weigh(cache(), rows(), w, nullptr); }); }
#define EVICT(why, ...) { auto e = evict(); e.__VA_ARGS__; \
    refused("evict: " #__VA_ARGS__, why, [&] { mit2hip::kv_evict(cache(), e, nullptr); }); }

int main() {
  CACHE("k, v and table", k = nullptr) CACHE("k, v and table", table = nullptr) CACHE("16-byte aligned", v = mem[21] + 8)
  CACHE("pages", pages = 0) CACHE("page_rows", page_rows = 3) CACHE("kv_heads", kv_heads = 0) CACHE("head_dim", head_dim = 80)
  CACHE("table_stride", table_stride = 0) CACHE("dtype", dtype = 3)
  ROWS("start and length", start = nullptr) ROWS("start and length", length = nullptr) ROWS("seqs", seqs = 65536) ROWS("rows", rows = 1u << 24)
  ROWS("4-byte aligned", start = at<int32_t>(1, 2))

  APPEND("k and v", k = nullptr) APPEND("k and v", v = nullptr) APPEND("q_out", q_out = nullptr) APPEND("rotary_dim", rotary_dim = 65)
  APPEND("theta", theta = 0.0) APPEND("q_heads", q_heads = 4097) APPEND("q_out's rows", q_out_head = 32) APPEND("q_out overlaps q", q_out = mem[5] + 128)
  APPEND("q_out overlaps k or v", q_out = mem[3]) APPEND("position", position = at<int32_t>(15, 1)) APPEND("aligned to their type", k = mem[3] + 1)
  APPEND("q_weight or k_weight", q_out = mem[7]) APPEND("q_weight or k_weight", q_out = mem[8])
  NORM("weight_dtype", weight_dtype = MIT2CFM_DTYPE_BF16) NORM("weight_dtype", weight_dtype = -1) NORM("eps", eps = 0.f) NORM("eps", eps = -1.f)
  NORM("eps", eps = NAN) NORM("eps", eps = INFINITY) NORM("aligned to their type", q_weight = mem[7] + 1)
  NORM("aligned to their type", k_weight = mem[8] + 2, n.weight_dtype = MIT2CFM_DTYPE_F32)
  NORM("q_weight or k_weight", q_weight = mem[6] + 1022) NORM("q_weight or k_weight", k_weight = mem[5] + 3968, n.k_weight_head = 128)

  ATTEND("q and out", q = nullptr) ATTEND("q and out", out = nullptr) ATTEND("q_heads", q_heads = 3) ATTEND("q_heads", q_heads = 0)
  ATTEND("scale", scale = INFINITY) ATTEND("mask_words", mask = at<uint32_t>(15)) ATTEND("mask must be 4-byte", mask = at<uint32_t>(15, 1), a.mask_words = 1)
  ATTEND("out overlaps q", out = mem[5] + 512) ATTEND("out's rows", out_row = 100) ATTEND("workspace", workspace = nullptr)
  ATTEND("workspace", workspace_bytes = 100) ATTEND("workspace must be 16", workspace = mem[9] + 4) ATTEND("aligned to their type", out = mem[6] + 1)
  PREFIX("groups", groups = 65536) PREFIX("group and shared", group = nullptr) PREFIX("group and shared", shared = nullptr)
  PREFIX("4-byte aligned", group = at<int32_t>(10, 1)) PREFIX("4-byte aligned", shared = at<int32_t>(11, 2)) PREFIX("4-byte aligned", lse = at<float>(12, 3))
  PREFIX("lse overlaps", lse = at<float>(5)) PREFIX("lse overlaps", lse = at<float>(6, 1020))

  WEIGH("must not be NULL", q = nullptr) WEIGH("must not be NULL", lse = nullptr) WEIGH("must not be NULL", weights = nullptr)
  WEIGH("must not be NULL", weights_out = nullptr) WEIGH("q_heads", q_heads = 5) WEIGH("scale", scale = NAN) WEIGH("decay", decay = INFINITY)
  WEIGH("mask_words", mask = at<uint32_t>(10)) WEIGH("mask_words", mask_words = 1u << 24) WEIGH("weight_stride", weight_stride = 0)
  WEIGH("weight_stride", weight_stride = (1u << 30) + 1) WEIGH("q must be aligned", q = mem[5] + 1) WEIGH("4-byte aligned", lse = at<float>(12, 2))
  WEIGH("4-byte aligned", weights = at<float>(13, 1)) WEIGH("4-byte aligned", weights_out = at<float>(14, 2)) WEIGH("4-byte aligned", position = at<int32_t>(15, 1))
  WEIGH("4-byte aligned", born = at<int32_t>(16, 1)) WEIGH("4-byte aligned", mask = at<uint32_t>(10, 1), w.mask_words = 1)
  WEIGH("weights_out overlaps weights", weights_out = at<float>(13, 4)) WEIGH("q, lse or mask", weights_out = at<float>(5, 512))
  WEIGH("q, lse or mask", weights_out = at<float>(12)) WEIGH("q, lse or mask", mask = at<uint32_t>(14, 4), w.mask_words = 1)
  WEIGH("born overlaps", born = at<int32_t>(13)) WEIGH("born overlaps", born = at<int32_t>(14, 28)) WEIGH("born overlaps", born = at<int32_t>(5))
  WEIGH("born overlaps", born = at<int32_t>(12)) WEIGH("born overlaps", born = at<int32_t>(15, 4))
  { auto r = rows(); r.rows = (1u << 24) - 1;
    auto w = weigh(); w.q_heads = 18;
    refused("weigh: rows * q_heads", "rows * q_heads", [&] { mit2hip::kv_weigh(cache(), r, w, nullptr); }); }

  EVICT("must not be NULL", length = nullptr) EVICT("must not be NULL", keep = nullptr) EVICT("must not be NULL", weights = nullptr)
  EVICT("must not be NULL", weights_out = nullptr) EVICT("must not be NULL", length_out = nullptr) EVICT("belong together", born_out = nullptr)
  EVICT("belong together", now = nullptr) EVICT("belong together", born = nullptr) EVICT("seqs must be", seqs = 65536) EVICT("layers in", layers = 0)
  EVICT("layers in", layers = 16385) EVICT("2^24", seqs = 65535, e.layers = 129) EVICT("weight_stride in", weight_stride = 0)
  EVICT("weight_stride in", weight_stride = (1u << 30) + 1) EVICT("multiple of 8", layer_stride = 516) EVICT("smaller than a layer", layer_stride = 504)
  EVICT("4-byte aligned", length = at<int32_t>(2, 1)) EVICT("4-byte aligned", keep = at<int32_t>(17, 2)) EVICT("4-byte aligned", weights = at<float>(13, 2))
  EVICT("4-byte aligned", weights_out = at<float>(14, 1)) EVICT("4-byte aligned", born = at<int32_t>(15, 2)) EVICT("4-byte aligned", born_out = at<int32_t>(16, 2))
  EVICT("4-byte aligned", now = at<int32_t>(18, 2)) EVICT("4-byte aligned", length_out = at<int32_t>(19, 2))
  EVICT("weights_out overlaps weights", weights_out = at<float>(13, 8)) EVICT("born_out overlaps born", born_out = at<int32_t>(15, 8))
  EVICT("overlap", born_out = at<int32_t>(13)) EVICT("overlap", born = at<int32_t>(14), e.born_out = at<int32_t>(14)) EVICT("overlap", now = at<int32_t>(14))
  EVICT("overlap", now = at<int32_t>(16)) EVICT("overlap", now = at<int32_t>(19)) EVICT("overlaps length, keep", keep = at<int32_t>(14))
  EVICT("overlaps length, keep", keep = at<int32_t>(19)) EVICT("overlaps length, keep", length_out = at<int32_t>(2, 4))
  EVICT("overlaps length, keep", length_out = at<int32_t>(13)) EVICT("overlaps length, keep", length_out = at<int32_t>(15))
  EVICT("overlaps length, keep", weights_out = at<float>(2)) EVICT("workspace", workspace = nullptr) EVICT("workspace", workspace_bytes = 100)
  EVICT("workspace must be 16", workspace = mem[9] + 8)

  std::printf("sizes %zu %zu %zu %zu\n", sizeof(mit2cfm_kv_norm), sizeof(mit2cfm_kv_prefix), sizeof(mit2cfm_kv_weigh), sizeof(mit2cfm_kv_evict));
  std::printf("offsets %zu %zu %zu %zu\n", offsetof(mit2cfm_kv_norm, eps), offsetof(mit2cfm_kv_prefix, lse), offsetof(mit2cfm_kv_weigh, born),
              offsetof(mit2cfm_kv_evict, workspace_bytes));
  std::printf("%d tried, %d wrong\n", tried, bad);
  return bad ? 1 : 0;
}
