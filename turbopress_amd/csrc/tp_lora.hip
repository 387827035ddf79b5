// Low-rank adapters of many requests beside a shared projection:
//
//   out[r] = y[r] + scale_i (x[r] A_i^T) B_i^T,  i = adapters[r]
//
// in two launches: a wave per (row, rank) for x A^T, a thread per output.
#include "tp_ops_common.h"

namespace tp {

struct LoraArgs {
  const void *x, *a, *b, *y;
  void* out;
  const int32_t* adapters;
  const float* scales;
  float* h;
  int64_t ldx, ldy, a_adapter, a_row, b_adapter, b_row, rows, k, n;
  int rank, count;
};

template <typename T>
__global__ void __launch_bounds__(256) lora_shrink_kernel(const LoraArgs p) {
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t row = at / p.rank;
  const int r = (int)(at - row * p.rank);
  if (row >= p.rows) return;
  const int i = p.adapters[row];
  if (i < 0 || i >= p.count) return;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* w = static_cast<const T*>(p.a) + i * p.a_adapter + r * p.a_row;
  float s = 0.0f;
  for (int64_t c = lane; c < p.k; c += 64) s += (float)x[c] * (float)w[c];
  s = reduce64<AddOp>(s);
  if (lane == 0) p.h[row * p.rank + r] = s;
}

template <typename T>
__global__ void __launch_bounds__(256) lora_expand_kernel(const LoraArgs p) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = at / p.n, c = at - row * p.n;
  if (row >= p.rows) return;
  const int i = p.adapters[row];
  const T base = static_cast<const T*>(p.y)[row * p.ldy + c];
  T* out = static_cast<T*>(p.out) + row * p.n + c;
  if (i < 0 || i >= p.count) {
    *out = base;
    return;
  }
  const T* w = static_cast<const T*>(p.b) + i * p.b_adapter + c * p.b_row;
  float s = 0.0f;
  for (int r = 0; r < p.rank; ++r) s += p.h[row * p.rank + r] * (float)w[r];
  *out = (T)((float)base + (p.scales ? p.scales[i] : 1.0f) * s);
}

template <typename T>
int launch_lora(const LoraArgs& p, hipStream_t s) {
  hipLaunchKernelGGL((lora_shrink_kernel<T>), dim3((uint32_t)((p.rows * p.rank + 3) / 4)), dim3(256), 0, s, p);
  hipLaunchKernelGGL((lora_expand_kernel<T>), dim3((uint32_t)((p.rows * p.n + 255) / 256)), dim3(256), 0, s, p);
  return launch_status();
}

}  // namespace tp

using namespace tp;

static bool lora_sizes_ok(int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count) {
  return rows >= 0 && rows <= (1 << 24) && k >= 1 && k <= (1 << 20) && n >= 1 && n <= (1 << 24) && rank >= 1 && rank <= 256 &&
         count >= 0 && count <= (1 << 20) && grid_fits((rows * rank + 3) / 4, 256) && grid_fits((rows * n + 255) / 256, 256);
}

extern "C" int64_t tp_lora_workspace_bytes(int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count) {
  return lora_sizes_ok(rows, k, n, rank, count) ? rows * rank * 4 : -1;
}

extern "C" int tp_lora_add(int dtype, int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count, const void* x,
                           int64_t ldx, const void* a, int64_t a_adapter, int64_t a_row, const void* b,
                           int64_t b_adapter, int64_t b_row, const int32_t* adapters, const float* scales,
                           const void* y, int64_t ldy, void* out, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  if (dtype != TP_F16 && dtype != TP_BF16) return TP_ERR_BAD_TYPE;
  if (!lora_sizes_ok(rows, k, n, rank, count)) return TP_ERR_BAD_DIMS;
  if (rows == 0) return TP_OK;
  if (!x || !y || !out || !adapters || (count && (!a || !b))) return TP_ERR_NULL_POINTER;
  if (!workspace || workspace_bytes < rows * rank * 4) return TP_ERR_WORKSPACE;
  LoraArgs p{x, a, b, y, out, adapters, scales, static_cast<float*>(workspace), ldx, ldy, a_adapter, a_row, b_adapter, b_row,
             rows, k, n, (int)rank, (int)count};
  return dtype == TP_F16 ? launch_lora<f16_t>(p, (hipStream_t)stream) : launch_lora<bf16_t>(p, (hipStream_t)stream);
}
