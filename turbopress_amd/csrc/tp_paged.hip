// Attention of one new token per sequence over a paged cache, with the running
// maximum and sum of a softmax:
//
//   m' = max(m, s_t),  l' = l e^(m - m') + e^(s_t - m'),  o' = o e^(m - m') + e^(s_t - m') v_t
//
// and two such states joined the same way.
#include "tp_ops_common.h"

#include <algorithm>

namespace tp {

// Where a running maximum starts: finite, so that a score of -infinity has
// probability e^-inf = 0 and not NaN, also where every score is -infinity.
constexpr float kLeastScore = -3.0e38f;

struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  const int32_t *block_table, *lengths;
  int64_t q_batch, q_head, kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  int64_t n_pages, table_width, window;
  int batch, hq, hkv, group, d, page_size;
  float scale;  // of the scores, in base 2
};

// A workgroup per (sequence, query head); each of its waves takes every fourth
// token, lane l columns 4 l .. 4 l + 3.
template <typename T>
__global__ void __launch_bounds__(256) paged_attention_kernel(const PagedArgs a) {
  __shared__ float part[4][258];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.y, h = blockIdx.x, kvh = h / a.group;
  const bool in = 4 * lane < a.d;
  int64_t len = a.lengths[b];
  len = min(max(len, (int64_t)0), a.table_width * a.page_size);
  const int64_t first = a.window > 0 ? max((int64_t)0, len - a.window) : 0;
  const int32_t* bt = a.block_table + (int64_t)b * a.table_width;
  float q[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0}, m = kLeastScore, l = 0.0f;
  if (in)
    for (int e = 0; e < 4; ++e)
      q[e] = (float)static_cast<const T*>(a.q)[b * a.q_batch + h * a.q_head + 4 * lane + e] * a.scale;
  for (int64_t t = first + wave; t < len; t += 4) {
    const int64_t page = bt[t / a.page_size], slot = t % a.page_size;
    if (page < 0 || page >= a.n_pages) continue;
    const T* k = static_cast<const T*>(a.k) + page * a.kc_page + slot * a.kc_slot + kvh * a.kc_head + 4 * lane;
    const T* v = static_cast<const T*>(a.v) + page * a.vc_page + slot * a.vc_slot + kvh * a.vc_head + 4 * lane;
    float s = 0.0f;
    if (in)
      for (int e = 0; e < 4; ++e) s = fmaf(q[e], (float)k[e], s);
    s = reduce64<AddOp>(s);
    const float m2 = fmaxf(m, s), keep = m == m2 ? 1.0f : exp2f(m - m2), p = exp2f(s - m2);
    l = l * keep + p;
    if (in)
      for (int e = 0; e < 4; ++e) o[e] = o[e] * keep + p * (float)v[e];
    m = m2;
  }
  for (int e = 0; e < 4; ++e) part[wave][4 * lane + e] = o[e];
  if (lane == 0) part[wave][256] = m, part[wave][257] = l;
  __syncthreads();
  float top = kLeastScore, total = 0.0f, y = 0.0f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][256]);
  for (int w = 0; w < 4; ++w) {
    const float f = part[w][257] > 0.0f ? exp2f(part[w][256] - top) : 0.0f;
    total += f * part[w][257];
    y += f * part[w][threadIdx.x];
  }
  if ((int)threadIdx.x < a.d)
    static_cast<T*>(a.out)[((int64_t)b * a.hq + h) * a.d + threadIdx.x] = (T)(total > 0.0f ? y / total : 0.0f);
}

bool paged_sizes_ok(int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  return batch >= 0 && batch <= 65535 && hq >= 1 && hkv >= 1 && hq <= 65536 && hq % hkv == 0 && d >= 8 && d <= 256 && d % 8 == 0;
}

}  // namespace tp

using namespace tp;

extern "C" int64_t tp_paged_attention_workspace_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  return paged_sizes_ok(batch, hq, hkv, d) ? 0 : -1;
}

extern "C" int tp_paged_attention(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d, const void* q,
                                  int64_t q_batch, int64_t q_head, const void* k_cache, const int64_t* kc,
                                  const void* v_cache, const int64_t* vc, int64_t n_pages, int64_t page_size,
                                  const int32_t* block_table, int64_t table_width, const int32_t* lengths,
                                  float scale, int64_t window, void* out, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (dtype != TP_F16 && dtype != TP_BF16) return TP_ERR_BAD_TYPE;
  if (!paged_sizes_ok(batch, hq, hkv, d) || n_pages < 0 || page_size < 1 || page_size > (1 << 24) || table_width < 0 ||
      table_width > (1 << 30) || window < 0)
    return TP_ERR_BAD_DIMS;
  if (batch == 0) return TP_OK;
  if (!q || !k_cache || !kc || !v_cache || !vc || !block_table || !lengths || !out) return TP_ERR_NULL_POINTER;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) return TP_ERR_MISALIGNED;
  if ((q_batch | q_head | kc[0] | kc[1] | kc[2] | vc[0] | vc[1] | vc[2]) & 7) return TP_ERR_MISALIGNED;
  if (((uintptr_t)block_table | (uintptr_t)lengths) & 3) return TP_ERR_MISALIGNED;
  PagedArgs a{};
  a.q = q, a.k = k_cache, a.v = v_cache, a.out = out, a.block_table = block_table, a.lengths = lengths;
  a.q_batch = q_batch, a.q_head = q_head;
  a.kc_page = kc[0], a.kc_slot = kc[1], a.kc_head = kc[2], a.vc_page = vc[0], a.vc_slot = vc[1], a.vc_head = vc[2];
  a.n_pages = n_pages, a.table_width = table_width, a.window = window;
  a.batch = (int)batch, a.hq = (int)hq, a.hkv = (int)hkv, a.group = (int)(hq / hkv), a.d = (int)d;
  a.page_size = (int)page_size, a.scale = scale * 1.44269504088896340736f;
  const dim3 grid((uint32_t)hq, (uint32_t)batch);
  if (dtype == TP_F16) hipLaunchKernelGGL((paged_attention_kernel<f16_t>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((paged_attention_kernel<bf16_t>), grid, dim3(256), 0, (hipStream_t)stream, a);
  return launch_status();
}
