// Attention over a paged cache: of one new token per sequence, and the entry points.
#include "tp_paged.h"

namespace tp {

bool paged_sizes_ok(int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  return batch >= 0 && batch <= (1 << 20) && hq >= 1 && hkv >= 1 && hq <= 65536 && hq % hkv == 0 && d >= 8 && d <= 256 && d % 8 == 0;
}

template <typename T>
int dispatch_paged(const PagedArgs& a, hipStream_t s) {
  switch (padded_d(a.d)) {
    case 64: launch_rows<T, 64, 1, 1, false>(a, s); break;
    case 96: launch_rows<T, 96, 1, 1, false>(a, s); break;
    case 128: launch_rows<T, 128, 1, 1, false>(a, s); break;
    case 192: launch_rows<T, 192, 1, 1, false>(a, s); break;
    default: launch_rows<T, 256, 1, 1, false>(a, s); break;
  }
  return launch_status();
}

}  // namespace tp

using namespace tp;

extern "C" int64_t tp_paged_attention_workspace_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  if (!paged_sizes_ok(batch, hq, hkv, d)) return -1;
  const int dp = padded_d(d);
  return (int64_t)device_cu_count() * 2 * kRowTile * (dp + 2) * (int64_t)sizeof(float);
}

extern "C" int64_t tp_paged_attention_counter_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  if (!paged_sizes_ok(batch, hq, hkv, d)) return -1;
  const int64_t tiles = (hq / hkv + kRowTile - 1) / kRowTile;
  return batch * hkv * tiles * (int64_t)sizeof(uint32_t);
}

// What the entry points share; of `a` ancestors, q_token, tokens and sinks are set.
static int paged_attention(PagedArgs a, int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d, const void* q,
                           int64_t q_batch, int64_t q_head, const void* k_cache, const int64_t* kc,
                           const void* v_cache, const int64_t* vc, int64_t n_pages, int64_t page_size,
                           const int32_t* block_table, int64_t table_width, const int32_t* lengths, float scale,
                           int64_t window, void* out, void* workspace, int64_t workspace_bytes, int64_t need,
                           void* counters, int64_t counter_bytes, int64_t count, void* stream) {
  if (dtype != TP_F16 && dtype != TP_BF16) return TP_ERR_BAD_TYPE;
  if (!paged_sizes_ok(batch, hq, hkv, d) || n_pages < 0 || n_pages > 0x7fffffff || page_size < 1 || page_size > (1 << 24) ||
      table_width < 0 || table_width > (1 << 30) || window < 0 || a.sinks < 0)
    return TP_ERR_BAD_DIMS;
  if (batch == 0) return TP_OK;
  if (!q || !kc || !vc || !lengths || !out || (n_pages > 0 && (!k_cache || !v_cache)) || (table_width > 0 && !block_table))
    return TP_ERR_NULL_POINTER;  // (empty tensors have no address)
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) return TP_ERR_MISALIGNED;
  if ((q_batch | q_head | kc[0] | kc[1] | kc[2] | vc[0] | vc[1] | vc[2]) & 7) return TP_ERR_MISALIGNED;
  if (((uintptr_t)block_table | (uintptr_t)lengths) & 3) return TP_ERR_MISALIGNED;
  if (!workspace || workspace_bytes < need || !counters || counter_bytes < count) return TP_ERR_WORKSPACE;
  if (((uintptr_t)workspace & 15) || ((uintptr_t)counters & 3)) return TP_ERR_MISALIGNED;
  a.q = q, a.k = k_cache, a.v = v_cache, a.out = out, a.block_table = block_table, a.lengths = lengths;
  a.parts = static_cast<float*>(workspace), a.counters = static_cast<uint32_t*>(counters);
  a.q_batch = q_batch, a.q_head = q_head;
  a.kc_page = kc[0], a.kc_slot = kc[1], a.kc_head = kc[2], a.vc_page = vc[0], a.vc_slot = vc[1], a.vc_head = vc[2];
  a.n_pages = n_pages, a.table_width = table_width, a.window = window;
  a.batch = (int)batch, a.hq = (int)hq, a.hkv = (int)hkv, a.group = (int)(hq / hkv), a.d = (int)d;
  a.row_groups = (int)(count / ((int64_t)sizeof(uint32_t) * batch * hkv));  // (a counter for each)
  a.page_size = (int)page_size, a.scale = scale * 1.44269504088896340736f;
  hipStream_t s = (hipStream_t)stream;
  if (a.tokens) return dtype == TP_F16 ? dispatch_tree_f16(a, s) : dispatch_tree_bf16(a, s);
  return dtype == TP_F16 ? dispatch_paged<f16_t>(a, s) : dispatch_paged<bf16_t>(a, s);
}

extern "C" int tp_paged_attention(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d, const void* q,
                                  int64_t q_batch, int64_t q_head, const void* k_cache, const int64_t* kc,
                                  const void* v_cache, const int64_t* vc, int64_t n_pages, int64_t page_size,
                                  const int32_t* block_table, int64_t table_width, const int32_t* lengths,
                                  float scale, int64_t window, void* out, void* workspace,
                                  int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream) {
  return tp_paged_attention_sinks(dtype, batch, hq, hkv, d, q, q_batch, q_head, k_cache, kc, v_cache, vc, n_pages, page_size,
                                  block_table, table_width, lengths, scale, window, 0, out, workspace, workspace_bytes, counters,
                                  counter_bytes, stream);
}

extern "C" int tp_paged_attention_sinks(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d, const void* q,
                                        int64_t q_batch, int64_t q_head, const void* k_cache, const int64_t* kc,
                                        const void* v_cache, const int64_t* vc, int64_t n_pages, int64_t page_size,
                                        const int32_t* block_table, int64_t table_width, const int32_t* lengths,
                                        float scale, int64_t window, int64_t sinks, void* out, void* workspace,
                                        int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream) {
  PagedArgs a{};
  a.sinks = sinks;
  return paged_attention(a, dtype, batch, hq, hkv, d, q, q_batch, q_head, k_cache, kc, v_cache, vc, n_pages, page_size,
                         block_table, table_width, lengths, scale, window, out, workspace, workspace_bytes,
                         tp_paged_attention_workspace_bytes(batch, hq, hkv, d), counters, counter_bytes,
                         tp_paged_attention_counter_bytes(batch, hq, hkv, d), stream);
}

static bool tree_sizes_ok(int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t d) {
  if (tokens < 1 || tokens > 64 || !paged_sizes_ok(batch, hq, hkv, d)) return false;
  const int64_t all = tokens * (hq / hkv), rows = kRowTile * tree_row_tiles(all, padded_d(d));
  return batch * hkv * ((all + rows - 1) / rows) <= (1 << 24);  // (the joins' workgroups)
}

extern "C" int64_t tp_paged_tree_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t d) {
  if (!tree_sizes_ok(batch, tokens, hq, hkv, d)) return -1;
  const int dp = padded_d(d), rows = kRowTile * tree_row_tiles(tokens * (hq / hkv), dp);
  return (int64_t)device_cu_count() * 2 * rows * (dp + 2) * (int64_t)sizeof(float);
}

extern "C" int64_t tp_paged_tree_attention_counter_bytes(int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t d) {
  if (!tree_sizes_ok(batch, tokens, hq, hkv, d)) return -1;
  const int64_t all = tokens * (hq / hkv), rows = kRowTile * tree_row_tiles(all, padded_d(d));
  return batch * hkv * ((all + rows - 1) / rows) * (int64_t)sizeof(uint32_t);
}

extern "C" int tp_paged_tree_attention(int dtype, int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t d,
                                       const void* q, int64_t q_batch, int64_t q_token, int64_t q_head,
                                       const void* k_cache, const int64_t* kc, const void* v_cache, const int64_t* vc,
                                       int64_t n_pages, int64_t page_size, const int32_t* block_table,
                                       int64_t table_width, const int32_t* lengths, const int64_t* ancestors,
                                       float scale, int64_t window, int64_t sinks, void* out, void* workspace,
                                       int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream) {
  if (dtype != TP_F16 && dtype != TP_BF16) return TP_ERR_BAD_TYPE;
  if (!tree_sizes_ok(batch, tokens, hq, hkv, d)) return TP_ERR_BAD_DIMS;
  if ((q_token & 7) || ((uintptr_t)ancestors & 7)) return TP_ERR_MISALIGNED;
  PagedArgs a{};
  a.ancestors = ancestors, a.q_token = q_token, a.tokens = (int)tokens, a.sinks = sinks;
  return paged_attention(a, dtype, batch, hq, hkv, d, q, q_batch, q_head, k_cache, kc, v_cache, vc, n_pages, page_size,
                         block_table, table_width, lengths, scale, window, out, workspace, workspace_bytes,
                         tp_paged_tree_attention_workspace_bytes(batch, tokens, hq, hkv, d), counters, counter_bytes,
                         tp_paged_tree_attention_counter_bytes(batch, tokens, hq, hkv, d), stream);
}
