// Log probabilities of given tokens, entropies and the most likely tokens of
// rows of logits: a workgroup per row.
#include "tp_ops_common.h"

namespace tp {

// The order of values: NaN above everything, negative zero with zero.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

struct LogprobArgs {
  const void* logits;
  const int64_t* tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  int64_t rows, vocab, ld;
  int top;
};

template <typename Op, int W>
__device__ __forceinline__ float block_reduce(float v, float (&s)[W]) {
  v = reduce64<Op>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < W; ++w) v = Op::of(v, s[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(1024) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int W = 16;
  __shared__ float s[W];
  __shared__ unsigned long long best;
  const T* x = static_cast<const T*>(a.logits) + blockIdx.x * a.ld;
  const int64_t row = blockIdx.x;
  float m = -INFINITY;
  for (int64_t i = threadIdx.x; i < a.vocab; i += 1024) m = MaxNanOp::of(m, (float)x[i]);
  m = block_reduce<MaxNanOp, W>(m, s);
  float count = 0.0f, rest = 0.0f, off = 0.0f;
  for (int64_t i = threadIdx.x; i < a.vocab; i += 1024) {
    const float f = (float)x[i], y = f - m;
    if (f == m) {
      count += 1.0f;
    } else {
      const float e = __expf(y);
      rest += e;
      if (e > 0.0f) off += e * y;
    }
  }
  count = block_reduce<AddOp, W>(count, s);
  rest = block_reduce<AddOp, W>(rest, s);
  off = block_reduce<AddOp, W>(off, s);
  const bool none = m == -INFINITY;  // nothing is possible
  const float more = count - 1.0f + rest, log_sum = m - m == 0.0f ? log1pf(more) : __builtin_nanf("");
  if (threadIdx.x == 0) {
    a.entropy[row] = none ? 0.0f : log_sum - off / (1.0f + more);
    if (a.tokens) {
      const int64_t t = a.tokens[row];
      a.logprobs[row] = t < 0 ? 0.0f : t >= a.vocab ? __builtin_nanf("") : none ? -INFINITY : (float)x[t] - m - log_sum;
    }
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    unsigned long long mine = 0;
    for (int64_t i = threadIdx.x; i < a.vocab; i += 1024) {
      const unsigned long long key = (unsigned long long)order_of((float)x[i]) << 32 | (uint32_t)~i;
      if (key < last && key > mine) mine = key;
    }
    if (threadIdx.x == 0) best = 0;
    __syncthreads();
    atomicMax(&best, mine);
    __syncthreads();
    last = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      const int64_t i = (uint32_t)~last;
      a.top_tokens[row * a.top + k] = i;
      a.top_logprobs[row * a.top + k] = none ? -INFINITY : (float)x[i] - m - log_sum;
    }
  }
}

}  // namespace tp

using namespace tp;

static bool logprob_sizes_ok(int64_t rows, int64_t vocab, int64_t top) {
  return rows >= 0 && rows <= (1 << 24) && vocab >= 1 && vocab <= (1 << 24) && top >= 0 && top <= 64 && top <= vocab;
}

extern "C" int64_t tp_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top) {
  return logprob_sizes_ok(rows, vocab, top) ? 16 : -1;
}

extern "C" int tp_token_logprobs(int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                                 const int64_t* tokens, float* logprobs, float* entropy, int top, float* top_logprobs,
                                 int64_t* top_tokens, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return TP_ERR_BAD_TYPE;
  if (!logprob_sizes_ok(rows, vocab, top)) return TP_ERR_BAD_DIMS;
  if (rows == 0) return TP_OK;
  if (!logits || !entropy || (tokens && !logprobs) || (top && (!top_logprobs || !top_tokens))) return TP_ERR_NULL_POINTER;
  LogprobArgs a{logits, tokens, logprobs, entropy, top_logprobs, top_tokens, rows, vocab, ld, top};
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((uint32_t)rows), block(1024);
  if (dtype == TP_F16) hipLaunchKernelGGL((token_logprobs_kernel<f16_t>), grid, block, 0, s, a);
  else if (dtype == TP_BF16) hipLaunchKernelGGL((token_logprobs_kernel<bf16_t>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((token_logprobs_kernel<float>), grid, block, 0, s, a);
  return launch_status();
}
