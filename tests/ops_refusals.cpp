// Calls the cache and beam operators with arguments that they must refuse
// before they touch a GPU, and prints the sizes of the argument structures.
// Exit status 1 when a call was not refused.
#include <cmath>
#include <cstddef>
#include <cstdio>
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

alignas(16) static char mem[64];
static int bad = 0, tried = 0;

static void refused(const char* what, const std::function<void()>& call) {
  ++tried;
  try {
    call();
  } catch (const std::invalid_argument&) {
    return;
  } catch (const std::exception& e) {
    std::printf("not refused as an argument: %s (%s)\n", what, e.what());
    ++bad;
    return;
  }
  std::printf("not refused: %s\n", what);
  ++bad;
}

static mit2cfm_kv_cache cache() {
  mit2cfm_kv_cache c{};
  c.k = c.v = mem;
  c.table = reinterpret_cast<int32_t*>(mem);
  c.pages = 4; c.page_rows = 16; c.kv_heads = 2; c.head_dim = 64; c.table_stride = 2;
  c.dtype = MIT2CFM_DTYPE_F16;
  return c;
}
static mit2cfm_kv_rows rows() {
  mit2cfm_kv_rows r{};
  r.start = r.length = reinterpret_cast<int32_t*>(mem);
  r.seqs = 1; r.rows = 2; r.max_length = 9;
  return r;
}
static mit2cfm_kv_append append() {
  mit2cfm_kv_append a{};
  a.k = a.v = a.q = mem;
  a.q_out = mem + 16;
  a.k_row = a.v_row = 128; a.k_head = a.v_head = a.q_head = a.q_out_head = 64;
  a.q_row = a.q_out_row = 256; a.q_heads = 4;
  a.rotary_dim = 64; a.theta = 10000.0;
  return a;
}
static mit2cfm_kv_attention attention() {
  mit2cfm_kv_attention a{};
  a.q = mem; a.out = mem + 16;
  a.q_row = a.out_row = 256; a.q_head = a.out_head = 64; a.q_heads = 4; a.scale = 0.125f;
  a.workspace = mem; a.workspace_bytes = ~0ull;
  return a;
}
static mit2cfm_beam_select select_args() {
  mit2cfm_beam_select a{};
  a.logits = mem; a.logits_row = 100; a.groups = 1; a.beams = 2; a.vocab = 100; a.count = 4;
  a.scores = reinterpret_cast<float*>(mem); a.stop_token = -1;
  a.scores_out = reinterpret_cast<float*>(mem + 16); a.parent_out = a.token_out = reinterpret_cast<int32_t*>(mem);
  a.workspace = mem; a.workspace_bytes = ~0ull;
  return a;
}
static mit2cfm_beam_reorder reorder_args() {
  mit2cfm_beam_reorder a{};
  a.groups = 1; a.beams = 2; a.layers = 2; a.layer_stride = 4 * 2 * 16 * 64;
  a.parent = a.length = reinterpret_cast<int32_t*>(mem); a.parent_stride = 2;
  a.table_out = reinterpret_cast<int32_t*>(mem + 16);
  a.state = reinterpret_cast<uint32_t*>(mem); a.state_out = reinterpret_cast<uint32_t*>(mem + 16); a.state_words = 3;
  a.token = reinterpret_cast<uint32_t*>(mem); a.place = reinterpret_cast<int32_t*>(mem);
  return a;
}

#define CACHE(...) { auto c = cache(); c.__VA_ARGS__; \
    refused("append: cache " #__VA_ARGS__, [&] { mit2hip::kv_append(c, rows(), append(), nullptr); }); \
    refused("attention: cache " #__VA_ARGS__, [&] { mit2hip::kv_attention(c, rows(), attention(), nullptr); }); \
    refused("reorder: cache " #__VA_ARGS__, [&] { mit2hip::beam_reorder(c, reorder_args(), nullptr); }); }
#define ROWS(...) { auto r = rows(); r.__VA_ARGS__; \
    refused("append: rows " #__VA_ARGS__, [&] { mit2hip::kv_append(cache(), r, append(), nullptr); }); \
    refused("attention: rows " #__VA_ARGS__, [&] { mit2hip::kv_attention(cache(), r, attention(), nullptr); }); }
#define APPEND(...) { auto a = append(); a.__VA_ARGS__; \
    refused("append: " #__VA_ARGS__, [&] { mit2hip::kv_append(cache(), rows(), a, nullptr); }); }
#define ATTEND(...) { auto a = attention(); a.__VA_ARGS__; \
    refused("attention: " #__VA_ARGS__, [&] { mit2hip::kv_attention(cache(), rows(), a, nullptr); }); }
#define SELECT(...) { auto a = select_args(); a.__VA_ARGS__; \
    refused("select: " #__VA_ARGS__, [&] { mit2hip::beam_select(a, nullptr); }); }
#define REORDER(...) { auto a = reorder_args(); a.__VA_ARGS__; \
    refused("reorder: " #__VA_ARGS__, [&] { mit2hip::beam_reorder(cache(), a, nullptr); }); }

int main() {
  CACHE(k = nullptr) CACHE(v = nullptr) CACHE(table = nullptr) CACHE(k = mem + 8) CACHE(v = mem + 4)
  CACHE(pages = 0) CACHE(pages = 1u << 31) CACHE(page_rows = 0) CACHE(page_rows = 24) CACHE(page_rows = 2048)
  CACHE(kv_heads = 0) CACHE(kv_heads = 1025) CACHE(head_dim = 0) CACHE(head_dim = 48) CACHE(head_dim = 512)
  CACHE(table_stride = 0) CACHE(table_stride = 1u << 27) CACHE(dtype = 3) CACHE(dtype = -1)
  CACHE(table_stride = (1u << 26) + 1) CACHE(table = reinterpret_cast<int32_t*>(mem + 2))
  ROWS(start = nullptr) ROWS(length = nullptr) ROWS(seqs = 65536) ROWS(rows = 1u << 24)
  ROWS(start = reinterpret_cast<int32_t*>(mem + 1)) ROWS(length = reinterpret_cast<int32_t*>(mem + 2))
  APPEND(k = nullptr) APPEND(v = nullptr) APPEND(k = mem + 1) APPEND(v = mem + 3) APPEND(q = mem + 1) APPEND(q_out = mem + 1)
  APPEND(q_out = nullptr) APPEND(q_heads = 0) APPEND(q_heads = 4097) APPEND(rotary_dim = 3) APPEND(rotary_dim = 66)
  APPEND(theta = 0.0) APPEND(theta = -1.0) APPEND(theta = NAN) APPEND(theta = INFINITY)
  APPEND(position = reinterpret_cast<int32_t*>(mem + 2))
  APPEND(q_out_head = 63) APPEND(q_out_row = 0) APPEND(q_out = mem, a.q_out_row = 512) APPEND(q_out = mem, a.q_out_head = 128)
  ATTEND(q = nullptr) ATTEND(out = nullptr) ATTEND(q = mem + 1) ATTEND(out = mem + 1) ATTEND(q_heads = 0) ATTEND(q_heads = 3)
  ATTEND(q_heads = 4098) ATTEND(scale = NAN) ATTEND(scale = INFINITY) ATTEND(out_head = 32) ATTEND(out_row = 63)
  ATTEND(mask = reinterpret_cast<uint32_t*>(mem)) ATTEND(mask = reinterpret_cast<uint32_t*>(mem), a.mask_words = 1u << 24)
  ATTEND(workspace = mem + 8) ATTEND(out = mem) ATTEND(mask = reinterpret_cast<uint32_t*>(mem + 2), a.mask_words = 1)
  { auto r = rows(); r.rows = (1u << 24) - 1;
    auto a = attention(); a.q_heads = 18;
    refused("attention: rows * q_heads", [&] { mit2hip::kv_attention(cache(), r, a, nullptr); }); }
  SELECT(logits = nullptr) SELECT(logits = mem + 2) SELECT(scores = nullptr) SELECT(scores_out = nullptr) SELECT(parent_out = nullptr)
  SELECT(token_out = nullptr) SELECT(dtype = 3) SELECT(dtype = -1) SELECT(beams = 0) SELECT(beams = 65) SELECT(vocab = 0)
  SELECT(vocab = (1u << 24) + 1) SELECT(count = 0) SELECT(count = 65) SELECT(count = 3, a.beams = 1, a.vocab = 2)
  SELECT(groups = (1u << 19) + 1) SELECT(stop_token = 100) SELECT(stop_token = -2) SELECT(finished = reinterpret_cast<int32_t*>(mem))
  SELECT(scores_out = reinterpret_cast<float*>(mem))
  SELECT(finished = a.token_out, a.finished_out = a.token_out, a.stop_token = 5) SELECT(scores = reinterpret_cast<float*>(mem + 2))
  SELECT(parent_out = reinterpret_cast<int32_t*>(mem + 1)) SELECT(finished_out = reinterpret_cast<int32_t*>(mem + 3))
  SELECT(workspace = nullptr) SELECT(workspace_bytes = 15) SELECT(workspace = mem + 8)
  REORDER(beams = 0) REORDER(beams = 65) REORDER(groups = (1u << 19) + 1) REORDER(layers = 0) REORDER(layers = 16385)
  REORDER(layer_stride = 4) REORDER(parent_stride = 1) REORDER(parent = nullptr) REORDER(length = nullptr) REORDER(table_out = nullptr)
  REORDER(table_out = reinterpret_cast<int32_t*>(mem)) REORDER(state_out = nullptr) REORDER(state_out = reinterpret_cast<uint32_t*>(mem))
  REORDER(state_words = 0) REORDER(state_words = 1u << 31) REORDER(state = nullptr) REORDER(place = nullptr)
  REORDER(parent = reinterpret_cast<int32_t*>(mem + 2)) REORDER(state = reinterpret_cast<uint32_t*>(mem + 1)) REORDER(place = reinterpret_cast<int32_t*>(mem + 2))
  std::printf("sizes %zu %zu %zu %zu %zu %zu\n", sizeof(mit2cfm_kv_cache), sizeof(mit2cfm_kv_rows), sizeof(mit2cfm_kv_append),
              sizeof(mit2cfm_kv_attention), sizeof(mit2cfm_beam_select), sizeof(mit2cfm_beam_reorder));
  std::printf("offsets %zu %zu %zu %zu %zu %zu\n", offsetof(mit2cfm_kv_cache, dtype), offsetof(mit2cfm_kv_rows, max_length),
              offsetof(mit2cfm_kv_append, theta), offsetof(mit2cfm_kv_attention, workspace_bytes),
              offsetof(mit2cfm_beam_select, workspace_bytes), offsetof(mit2cfm_beam_reorder, place));
  std::printf("%d tried, %d not refused\n", tried, bad);
  return bad ? 1 : 0;
}
