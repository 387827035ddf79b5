// Attention of a tree of drafted tokens of each sequence over a paged cache: a
// workgroup per (sequence, drafted token, query head), a wave per cached token.
#include "tp_ops_common.h"

namespace tp {

constexpr float kTreeLeast = -3.0e38f;

struct TreeArgs {
  const void *q, *k, *v;
  void* out;
  const int32_t *block_table, *lengths;
  const int64_t* ancestors;
  int64_t q_batch, q_token, q_head, kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  int64_t n_pages, table_width, window, sinks;
  int batch, tokens, hq, hkv, d, page_size;
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(256) tree_attention_kernel(const TreeArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head = blockIdx.x % a.hq;
  const int64_t bt = blockIdx.x / a.hq;
  const int b = (int)(bt / a.tokens), i = (int)(bt % a.tokens);
  const int kvh = head / (a.hq / a.hkv);
  const int64_t len = min(max(a.lengths[b], 0), 0x7fffe000);
  auto bits_of = [&](int j) { return a.ancestors ? (uint64_t)a.ancestors[(int64_t)b * a.tokens + j] : ~0ull >> (63 - j); };
  const uint64_t bits = bits_of(i) & (~0ull >> (64 - a.tokens));
  const int64_t position = len + __builtin_popcountll(bits) - 1;
  const int64_t end = min(len + a.tokens, a.table_width * a.page_size);
  const T* q = static_cast<const T*>(a.q) + b * a.q_batch + i * a.q_token + head * a.q_head;
  float qf[4], o[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) qf[e] = lane + 64 * e < a.d ? (float)q[lane + 64 * e] : 0.0f;
  float m = kTreeLeast, l = 0.0f;
  for (int64_t t = wave; t < end; t += 4) {
    int64_t place = t;
    if (t >= len) {
      const int j = (int)(t - len);
      if (!(bits >> j & 1)) continue;
      place = len + __builtin_popcountll(bits_of(j) & (~0ull >> (64 - a.tokens))) - 1;
    }
    if (a.window > 0 && place <= position - a.window && place >= a.sinks) continue;
    const int64_t page = a.block_table[b * a.table_width + t / a.page_size], slot = t % a.page_size;
    if (page < 0 || page >= a.n_pages) continue;
    const T* k = static_cast<const T*>(a.k) + page * a.kc_page + slot * a.kc_slot + kvh * a.kc_head;
    const T* v = static_cast<const T*>(a.v) + page * a.vc_page + slot * a.vc_slot + kvh * a.vc_head;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 64 * e < a.d) s += qf[e] * (float)k[lane + 64 * e];
    s = reduce64<AddOp>(s) * a.scale;
    const float top = fmaxf(m, s), keep = __builtin_amdgcn_exp2f(m - top), p = __builtin_amdgcn_exp2f(s - top);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 64 * e < a.d) o[e] = o[e] * keep + p * (float)v[lane + 64 * e];
  }
  __shared__ float ms[4], ls[4], os[4][256];
  if (lane == 0) ms[wave] = m, ls[wave] = l;
#pragma unroll
  for (int e = 0; e < 4; ++e) os[wave][lane + 64 * e] = o[e];
  __syncthreads();
  const int c = threadIdx.x;
  if (c >= a.d) return;
  const float top = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
  float sum = 0.0f, y = 0.0f;
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(ms[w] - top);
    sum += f * ls[w];
    y += f * os[w][c];
  }
  static_cast<T*>(a.out)[(bt * a.hq + head) * a.d + c] = (T)(sum == 0.0f ? 0.0f : y / sum);
}

}  // namespace tp

using namespace tp;

static bool tree_sizes_ok(int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t d) {
  return batch >= 0 && batch <= (1 << 20) && tokens >= 1 && tokens <= 64 && hq >= 1 && hkv >= 1 && hq <= 65536 &&
         hq % hkv == 0 && d >= 8 && d <= 256 && d % 8 == 0 && grid_fits(batch * tokens * hq, 256);
}

extern "C" int64_t tp_paged_tree_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t d) {
  return tree_sizes_ok(batch, tokens, hq, hkv, d) ? 16 : -1;
}

extern "C" int64_t tp_paged_tree_attention_counter_bytes(int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t d) {
  return tree_sizes_ok(batch, tokens, hq, hkv, d) ? 16 : -1;
}

extern "C" int tp_paged_tree_attention(int dtype, int64_t batch, int64_t tokens, int64_t hq, int64_t hkv, int64_t d,
                                       const void* q, int64_t q_batch, int64_t q_token, int64_t q_head,
                                       const void* k_cache, const int64_t* kc, const void* v_cache, const int64_t* vc,
                                       int64_t n_pages, int64_t page_size, const int32_t* block_table,
                                       int64_t table_width, const int32_t* lengths, const int64_t* ancestors,
                                       float scale, int64_t window, int64_t sinks, void* out, void* workspace,
                                       int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream) {
  if (dtype != TP_F16 && dtype != TP_BF16) return TP_ERR_BAD_TYPE;
  if (!tree_sizes_ok(batch, tokens, hq, hkv, d) || n_pages < 0 || n_pages > 0x7fffffff || page_size < 1 ||
      page_size > (1 << 24) || table_width < 0 || table_width > (1 << 30) || window < 0 || sinks < 0)
    return TP_ERR_BAD_DIMS;
  if (batch == 0) return TP_OK;
  if (!q || !kc || !vc || !lengths || !out || (n_pages > 0 && (!k_cache || !v_cache)) || (table_width > 0 && !block_table))
    return TP_ERR_NULL_POINTER;
  TreeArgs a{};
  a.q = q, a.k = k_cache, a.v = v_cache, a.out = out, a.block_table = block_table, a.lengths = lengths, a.ancestors = ancestors;
  a.q_batch = q_batch, a.q_token = q_token, a.q_head = q_head;
  a.kc_page = kc[0], a.kc_slot = kc[1], a.kc_head = kc[2], a.vc_page = vc[0], a.vc_slot = vc[1], a.vc_head = vc[2];
  a.n_pages = n_pages, a.table_width = table_width, a.window = window, a.sinks = sinks;
  a.batch = (int)batch, a.tokens = (int)tokens, a.hq = (int)hq, a.hkv = (int)hkv, a.d = (int)d, a.page_size = (int)page_size;
  a.scale = scale * 1.44269504088896340736f;
  const dim3 grid((uint32_t)(batch * tokens * hq));
  if (dtype == TP_F16) hipLaunchKernelGGL((tree_attention_kernel<f16_t>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((tree_attention_kernel<bf16_t>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return launch_status();
}
