// Rotary positions of queries and keys, alone or with keys and values written
// into a paged cache.  The pair (a, b) of index i of a head becomes
//
//   (a c_i - b s_i, b c_i + a s_i)
//
// with the position's cosines and sines from a table (fp32, made in 64 bits
// once: an angle position * frequency formed in fp32 is off by up to 2^-24 of
// the position, 0.008 at position 131072).  Each element is read and written
// once; 3 flops per element: bound by HBM, or by latency for a few tokens.
// 2047 tokens of 32 + 8 + 8 heads of 128 into the cache 7.8 us (34 MB, part of
// them out of the memory-side cache), one token of 4 sequences 2.7.
#include "tp_ops_common.h"

#include <algorithm>

namespace tp {

struct RotaryArgs {
  const void *q, *k, *v;
  void *q_out, *k_out, *k_cache, *v_cache;
  const float* table;
  const int64_t* positions;
  const int32_t *block_table, *sequences;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  int64_t tokens, n_positions, n_pages, page_size, table_width, n_sequences;
  int hq, hk, hv, d, rd, interleaved;
  int units, rot_units;  // of 2 V elements per head; the first rot_units turn
};

// Stored past the caches where that is whole 16-byte pieces.
template <typename P, typename T>
__device__ __forceinline__ void store_once(T* p, const P& v) {
  if constexpr (sizeof(P) % 16 == 0) {
    u32x4 w[sizeof(P) / 16];
    __builtin_memcpy(w, &v, sizeof(v));
#pragma unroll
    for (int i = 0; i < (int)sizeof(P) / 16; ++i) __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4_any*>(p) + i);
  } else {
    __builtin_memcpy(p, &v, sizeof(v));
  }
}

// A thread per (token, head, unit of 2 V elements): V pairs, or 2 V elements
// that are copied.  Units of the half layout take V elements of either half.
template <typename T, int V>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  struct Part {
    T v[V];
  };
  const int heads = a.hq + a.hk + a.hv;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t per = (int64_t)heads * a.units;
  const int64_t t = at / per;
  if (t >= a.tokens) return;
  const int rest = (int)(at - t * per);
  int head = rest / a.units;
  const int u = rest - head * a.units;

  const T* src;
  T* dst;
  const int64_t p = a.positions[t];
  const bool padding = p < 0, past = p >= a.n_positions;
  const bool is_q = head < a.hq, is_v = head >= a.hq + a.hk;
  if (is_q) {
    src = static_cast<const T*>(a.q) + t * a.q_token + head * a.q_head;
    dst = static_cast<T*>(a.q_out) + (t * a.hq + head) * a.d;
  } else {
    head -= is_v ? a.hq + a.hk : a.hq;
    src = is_v ? static_cast<const T*>(a.v) + t * a.v_token + head * a.v_head
               : static_cast<const T*>(a.k) + t * a.k_token + head * a.k_head;
    if (a.k_cache) {
      if (padding || past) return;
      const int64_t seq = a.sequences ? (int64_t)a.sequences[t] : t;
      const int64_t col = p / a.page_size;
      if (seq < 0 || seq >= a.n_sequences || col >= a.table_width) return;
      const int64_t page = a.block_table[seq * a.table_width + col], slot = p - col * a.page_size;
      if (page < 0 || page >= a.n_pages) return;
      dst = is_v ? static_cast<T*>(a.v_cache) + page * a.vc_page + slot * a.vc_slot + head * a.vc_head
                 : static_cast<T*>(a.k_cache) + page * a.kc_page + slot * a.kc_slot + head * a.kc_head;
    } else {
      dst = static_cast<T*>(a.k_out) + (t * a.hk + head) * a.d;
    }
  }

  const bool turn = !is_v && u < a.rot_units;
  const bool halves = turn && !a.interleaved;
  const int first = halves ? u * V : u * 2 * V, second = halves ? first + a.rd / 2 : first + V;
  Part x, y;
  __builtin_memcpy(&x, src + first, sizeof(x));
  __builtin_memcpy(&y, src + second, sizeof(y));
  if (padding || past) {
    const T fill = (T)(past ? __builtin_nanf("") : 0.0f);
#pragma unroll
    for (int e = 0; e < V; ++e) x.v[e] = y.v[e] = fill;
  } else if (turn) {
    const float* cs = a.table + p * a.rd + u * V;
    float c[V], s[V];
    __builtin_memcpy(c, cs, sizeof(c));
    __builtin_memcpy(s, cs + a.rd / 2, sizeof(s));
    float f[2 * V];
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (float)x.v[e], f[V + e] = (float)y.v[e];
    auto pair = [&](float& p0, float& p1, int e) __attribute__((always_inline)) {
      const float x0 = p0, x1 = p1;
      p0 = x0 * c[e] - x1 * s[e];
      p1 = x1 * c[e] + x0 * s[e];
    };
    if (a.interleaved) {
#pragma unroll
      for (int e = 0; e < V; ++e) pair(f[2 * e], f[2 * e + 1], e);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) pair(f[e], f[V + e], e);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) x.v[e] = (T)f[e], y.v[e] = (T)f[V + e];
  }
  store_once(dst + first, x);
  store_once(dst + second, y);
}

template <typename T>
int launch_rotary(RotaryArgs a, hipStream_t s) {
  // the widest unit that cuts the halves and the copied rest evenly
  int v = 8;
  while (v > 1 && ((a.rd / 2) % v || (a.d - a.rd) % (2 * v))) v /= 2;
  a.units = a.d / (2 * v), a.rot_units = a.rd / (2 * v);
  const int64_t each = (int64_t)(a.hq + a.hk + a.hv) * a.units;  // units of a token
  // (a launch holds less than 2^32 threads; a token's are counted in 31 bits, for
  // unsigned division made 32768 tokens of 12 heads of 64 2 % slower)
  if (each > 0x7fffffff || a.tokens > 0xffffff00ll / each) return TP_ERR_BAD_DIMS;
  const int64_t blocks = (a.tokens * each + 255) / 256;
  const dim3 grid((uint32_t)blocks), block(256);
  if (v == 8) hipLaunchKernelGGL((rotary_kernel<T, 8>), grid, block, 0, s, a);
  else if (v == 4) hipLaunchKernelGGL((rotary_kernel<T, 4>), grid, block, 0, s, a);
  else if (v == 2) hipLaunchKernelGGL((rotary_kernel<T, 2>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((rotary_kernel<T, 1>), grid, block, 0, s, a);
  return launch_status();
}

}  // namespace tp

using namespace tp;

extern "C" int tp_rotary(int dtype, int64_t tokens, int64_t hq, int64_t hk, int64_t d, int64_t rotary_dim,
                         int interleaved, const void* q, int64_t q_token, int64_t q_head, const void* k,
                         int64_t k_token, int64_t k_head, const float* table, int64_t n_positions,
                         const int64_t* positions, void* q_out, void* k_out, const void* v, int64_t v_token,
                         int64_t v_head, void* k_cache, const int64_t* kc, void* v_cache, const int64_t* vc,
                         int64_t n_pages, int64_t page_size, const int32_t* block_table, int64_t table_width,
                         int64_t n_sequences, const int32_t* sequences, void* stream) {
  if (!dtype_ok(dtype)) return TP_ERR_BAD_TYPE;
  if (tokens < 0 || hq < 0 || hk < 0 || hq > 65536 || hk > 65536 || d < 2 || d > 65536 || (d & 1) || rotary_dim < 2 ||
      rotary_dim > d || (rotary_dim & 1) || n_positions < 0 || tokens > ((int64_t)1 << 40))
    return TP_ERR_BAD_DIMS;
  if (tokens == 0 || hq + hk == 0) return TP_OK;
  if (!table || !positions || (hq && (!q || !q_out))) return TP_ERR_NULL_POINTER;
  RotaryArgs a{};
  if (k_cache) {
    if (!hk || n_pages < 0 || page_size < 1 || table_width < 0 || n_sequences < 0) return TP_ERR_BAD_DIMS;
    if (!k || !v || !v_cache || !kc || !vc || (table_width > 0 && n_sequences > 0 && !block_table)) return TP_ERR_NULL_POINTER;
    a.hv = (int)hk;
    a.kc_page = kc[0], a.kc_slot = kc[1], a.kc_head = kc[2], a.vc_page = vc[0], a.vc_slot = vc[1], a.vc_head = vc[2];
  } else if (hk && (!k || !k_out)) {
    return TP_ERR_NULL_POINTER;
  }
  const uintptr_t mask = dtype_bytes(dtype) - 1;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)k_cache |
        (uintptr_t)v_cache) & mask) || (((uintptr_t)table | (uintptr_t)block_table | (uintptr_t)sequences) & 3) ||
      ((uintptr_t)positions & 7))
    return TP_ERR_MISALIGNED;
  a.q = q, a.k = k, a.v = v, a.q_out = q_out, a.k_out = k_out, a.k_cache = k_cache, a.v_cache = v_cache;
  a.table = table, a.positions = positions, a.block_table = block_table, a.sequences = sequences;
  a.q_token = q_token, a.q_head = q_head, a.k_token = k_token, a.k_head = k_head, a.v_token = v_token, a.v_head = v_head;
  a.tokens = tokens, a.n_positions = n_positions, a.n_pages = n_pages, a.page_size = page_size;
  a.table_width = table_width, a.n_sequences = n_sequences;
  a.hq = (int)hq, a.hk = (int)hk, a.d = (int)d, a.rd = (int)rotary_dim, a.interleaved = interleaved != 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TP_F16) return launch_rotary<f16_t>(a, s);
  if (dtype == TP_BF16) return launch_rotary<bf16_t>(a, s);
  return launch_rotary<float>(a, s);
}
