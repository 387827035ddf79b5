// Product of e4m3 activations and weights with scales per 128 columns:
//
//   y[i, j] = sum_b a_scales[i, b] w_scales[j / 128, b] sum_{c in block b} a[i, c] w[j, c]  (+ bias[j])
#include "tp_ops_common.h"

#include <algorithm>

namespace tp {

struct Fp8Args {
  const uint8_t *a, *w;
  const float *sa, *sw;
  const void* bias;
  void* y;
  int64_t lda, ldw, ldy, m, n;
  int k, kb;
};

template <typename T>
__global__ void __launch_bounds__(256) fp8_linear_kernel(const Fp8Args a) {
  const int64_t j = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int64_t i = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6);
  if (i >= a.m || j >= a.n) return;
  const uint8_t* ar = a.a + i * a.lda;
  const uint8_t* wr = a.w + j * a.ldw;
  float y = 0.0f;
  for (int b = 0; b < a.kb; ++b) {
    float part = 0.0f;
    for (int c = 128 * b; c < min(a.k, 128 * b + 128); ++c)
      part = fmaf(__builtin_amdgcn_cvt_f32_fp8(ar[c], 0), __builtin_amdgcn_cvt_f32_fp8(wr[c], 0), part);
    y = fmaf(part, a.sa[i * a.kb + b] * a.sw[(j >> 7) * a.kb + b], y);
  }
  if (a.bias) y += (float)static_cast<const T*>(a.bias)[j];
  static_cast<T*>(a.y)[i * a.ldy + j] = (T)y;
}

template <typename T>
int launch_fp8(const Fp8Args& a, hipStream_t s) {
  hipLaunchKernelGGL((fp8_linear_kernel<T>), dim3((uint32_t)((a.n + 63) / 64), (uint32_t)((a.m + 3) / 4)), dim3(256), 0, s, a);
  return launch_status();
}

bool fp8_sizes_ok(int64_t m, int64_t n, int64_t k) {
  return m >= 0 && n >= 0 && k >= 1 && m <= 65535 * 4 && n <= (1 << 28) && k <= (1 << 20);
}

}  // namespace tp

using namespace tp;

extern "C" int64_t tp_fp8_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  return fp8_sizes_ok(m, n, k) ? 0 : -1;
}

extern "C" int tp_fp8_linear(int dtype, int64_t m, int64_t n, int64_t k, const uint8_t* a, int64_t lda,
                             const float* a_scales, const uint8_t* w, int64_t ldw, const float* w_scales,
                             const void* bias, void* y, int64_t ldy, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  if (!dtype_ok(dtype)) return TP_ERR_BAD_TYPE;
  if (!fp8_sizes_ok(m, n, k) || lda < k || ldw < k || ldy < n) return TP_ERR_BAD_DIMS;
  if (m == 0 || n == 0) return TP_OK;
  if (!a || !a_scales || !w || !w_scales || !y) return TP_ERR_NULL_POINTER;
  const uintptr_t mask = dtype_bytes(dtype) - 1;
  if ((((uintptr_t)a_scales | (uintptr_t)w_scales) & 3) || (((uintptr_t)bias | (uintptr_t)y) & mask))
    return TP_ERR_MISALIGNED;
  const int64_t need = tp_fp8_workspace_bytes(m, n, k);
  if (need > 0 && (!workspace || workspace_bytes < need)) return TP_ERR_WORKSPACE;
  Fp8Args g{a, w, a_scales, w_scales, bias, y, lda, ldw, ldy, m, n, (int)k, (int)((k + 127) / 128)};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TP_F16) return launch_fp8<f16_t>(g, s);
  if (dtype == TP_BF16) return launch_fp8<bf16_t>(g, s);
  return launch_fp8<float>(g, s);
}
