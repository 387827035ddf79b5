// Root-mean-square norm of rows, with the residual's addition, its output in
// the input's type or in 8-bit floating point with scales:
//
//   h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight
//   scale = max(max |y| / 448, 2^-126),  code = e4m3(y / scale)
//
// One pass: a row's h stays in registers (fp32) between its sum of squares and
// its output, so x and the residual are read once and h, y (or codes) written
// once; the weight comes from L2.  Nothing is computed to speak of (4 flops per
// element): many rows are bound by HBM, a few by the latency of load, reduction
// and store.
#include "tp_ops_common.h"

#include <algorithm>

namespace tp {

struct NormArgs {
  const void* x;
  const void* residual;
  const void* weight;
  void* y;
  uint8_t* codes;
  float* scales;
  void* h;
  int64_t x_outer, x_inner, r_outer, r_inner, ldc, rows;
  int inner, d, nvec, nblocks, waves_per_row;
  float eps;
};

enum NormOut { kSame = 0, kFp8Block = 1, kFp8Row = 2 };

constexpr float kE4m3Max = 448.0f;
constexpr float kLeastScale = 0x1p-126f;

// Elements [8 i, 8 i + 8) of a row of d, zeros past its end.
template <typename T>
__device__ __forceinline__ Vec<T> load_row8(const T* row, int i, int d) {
  if (8 * i + 8 <= d) return load8(row + 8 * i);
  Vec<T> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = 8 * i + e < d ? row[8 * i + e] : (T)0.0f;
  return r;
}

template <typename T>
__device__ __forceinline__ void store_row8(T* row, int i, int d, const Vec<T>& r) {
  if (8 * i + 8 <= d) {
    store8(row + 8 * i, r);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (8 * i + e < d) row[8 * i + e] = r.v[e];
}

// 8 values as e4m3 (v_cvt rounds to nearest even; a NaN stays one, |v| <= 448
// up to rounding, so nothing overflows).
__device__ __forceinline__ u32x2 to_e4m3(const float* v) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  return u32x2{(uint32_t)lo, (uint32_t)hi};
}

__device__ __forceinline__ float max_abs8(const float* v) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) m = MaxNanOp::of(m, fabsf(v[e]));
  return m;
}

__device__ __forceinline__ float scale_of(float amax) { return MaxNanOp::of(amax / kE4m3Max, kLeastScale); }

__device__ __forceinline__ size_t row_offset(int64_t row, int inner, int64_t outer_stride, int64_t inner_stride) {
  const int64_t o = row / inner;
  return (size_t)(o * outer_stride + (row - o * inner) * inner_stride);
}

// Over the lanes that hold one row: 16, 32 or 64 lanes of a wave, or
// waves_per_row waves of the workgroup (`slots`: an LDS word per wave).
template <typename Op, int SUB>
__device__ __forceinline__ float reduce_row(float v, int wpr, float* slots) {
  v = reduce16<Op>(v);
  if constexpr (SUB >= 32) v = combine16<Op>(v);
  if constexpr (SUB >= 64) {
    v = combine32<Op>(v);
    if (wpr > 1) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) slots[wave] = v;
      __syncthreads();
      const int first = wave & ~(wpr - 1);
      v = slots[first];
      for (int w = 1; w < wpr; ++w) v = Op::of(v, slots[first + w]);
    }
  }
  return v;
}

// A row per SUB lanes (SUB < 64) or per waves_per_row waves (SUB = 64), VPT
// vectors of 8 elements per lane.
template <typename T, int OUT, int SUB, int VPT>
__global__ void __launch_bounds__(512) rms_norm_kernel(const NormArgs a) {
  __shared__ float slots[32];
  const int wpr = SUB < 64 ? 1 : a.waves_per_row;
  const int lanes = SUB < 64 ? SUB : 64 * wpr;  // that hold one row
  const int i0 = (int)threadIdx.x & (lanes - 1);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / lanes) + (int)threadIdx.x / lanes;
  const bool live = row < a.rows;
  const int64_t rrow = live ? row : a.rows - 1;  // (idle lanes follow a row along, for the barriers)
  const T* x = static_cast<const T*>(a.x) + row_offset(rrow, a.inner, a.x_outer, a.x_inner);
  const T* weight = static_cast<const T*>(a.weight);

  float h[VPT][8];
  Vec<T> xv[VPT], wv[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j)
    if (i0 + j * lanes < a.nvec) xv[j] = load_row8(x, i0 + j * lanes, a.d);
  if (a.residual) {
    const T* res = static_cast<const T*>(a.residual) + row_offset(rrow, a.inner, a.r_outer, a.r_inner);
    Vec<T> rv[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (i0 + j * lanes < a.nvec) rv[j] = load_row8(res, i0 + j * lanes, a.d);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (i0 + j * lanes < a.nvec) wv[j] = load_row8(weight, i0 + j * lanes, a.d);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        h[j][e] = i0 + j * lanes < a.nvec ? (float)xv[j].v[e] + (float)rv[j].v[e] : 0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (i0 + j * lanes < a.nvec) wv[j] = load_row8(weight, i0 + j * lanes, a.d);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] = i0 + j * lanes < a.nvec ? (float)xv[j].v[e] : 0.0f;
  }

  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(h[j][e], h[j][e], sum);
  sum = reduce_row<AddOp, SUB>(sum, wpr, slots);
  const float inv = 1.0f / sqrtf(sum / (float)a.d + a.eps);

  if (a.h && live) {
    T* hr = static_cast<T*>(a.h) + (size_t)row * a.d;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (i0 + j * lanes < a.nvec) {
        Vec<T> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = (T)h[j][e];
        store_row8(hr, i0 + j * lanes, a.d, o);
      }
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) h[j][e] = i0 + j * lanes < a.nvec ? h[j][e] * inv * (float)wv[j].v[e] : 0.0f;

  if constexpr (OUT == kSame) {
    T* y = static_cast<T*>(a.y) + (size_t)row * a.d;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (live && i0 + j * lanes < a.nvec) {
        Vec<T> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = (T)h[j][e];
        store_row8(y, i0 + j * lanes, a.d, o);
      }
  } else {
    float s_row = 0.0f;
    if constexpr (OUT == kFp8Row) {
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < VPT; ++j) m = MaxNanOp::of(m, max_abs8(h[j]));
      s_row = scale_of(reduce_row<MaxNanOp, SUB>(m, wpr, slots + 16));
      if (live && i0 == 0) a.scales[row] = s_row;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = i0 + j * lanes;
      float s = s_row;
      if constexpr (OUT == kFp8Block) {  // 16 lanes hold a block of 128
        s = scale_of(reduce16<MaxNanOp>(max_abs8(h[j])));
        if (live && i < a.nvec && (i & 15) == 0) a.scales[(size_t)row * a.nblocks + (i >> 4)] = s;
      }
      const float is = 1.0f / s;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] *= is;
      if (live && i < a.nvec) *reinterpret_cast<u32x2*>(a.codes + (size_t)row * a.ldc + 8 * i) = to_e4m3(h[j]);
    }
  }
}

// Rows too long for the registers of 512 threads: a workgroup per row, which
// reads it again for each of its passes (from L2: a row is at most a few MB).
template <typename T, int OUT>
__global__ void __launch_bounds__(1024) rms_norm_long_kernel(const NormArgs a) {
  __shared__ float slots[32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row_offset(row, a.inner, a.x_outer, a.x_inner);
  const T* res = a.residual ? static_cast<const T*>(a.residual) + row_offset(row, a.inner, a.r_outer, a.r_inner) : nullptr;
  const T* weight = static_cast<const T*>(a.weight);
  const int tid = threadIdx.x;
  auto load_h = [&](int i, float* h) __attribute__((always_inline)) {
    const Vec<T> xv = load_row8(x, i, a.d);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (float)xv.v[e];
    if (res) {
      const Vec<T> rv = load_row8(res, i, a.d);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] += (float)rv.v[e];
    }
  };
  float sum = 0.0f;
  for (int i = tid; i < a.nvec; i += 1024) {
    float h[8];
    load_h(i, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(h[e], h[e], sum);
  }
  sum = reduce_row<AddOp, 64>(sum, 16, slots);
  const float inv = 1.0f / sqrtf(sum / (float)a.d + a.eps);
  auto load_y = [&](int i, float* h) __attribute__((always_inline)) {
    load_h(i, h);
    const Vec<T> wv = load_row8(weight, i, a.d);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = h[e] * inv * (float)wv.v[e];
  };
  float s = 0.0f;
  if constexpr (OUT == kFp8Row) {
    float m = 0.0f;
    for (int i = tid; i < a.nvec; i += 1024) {
      float y[8];
      load_y(i, y);
      m = MaxNanOp::of(m, max_abs8(y));
    }
    s = scale_of(reduce_row<MaxNanOp, 64>(m, 16, slots + 16));
    if (tid == 0) a.scales[row] = s;
  }
  // (whole rows of 16 lanes stay together, for the block's maximum)
  const int end = OUT == kFp8Block ? (a.nvec + 15) & ~15 : a.nvec;
  for (int i = tid; i < end; i += 1024) {
    const bool in = i < a.nvec;
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (in) {
      if (a.h) {
        float h[8];
        load_h(i, h);
        Vec<T> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = (T)h[e];
        store_row8(static_cast<T*>(a.h) + (size_t)row * a.d, i, a.d, o);
      }
      load_y(i, y);
    }
    if constexpr (OUT == kSame) {
      Vec<T> o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = (T)y[e];
      store_row8(static_cast<T*>(a.y) + (size_t)row * a.d, i, a.d, o);
    } else {
      if constexpr (OUT == kFp8Block) {
        s = scale_of(reduce16<MaxNanOp>(max_abs8(y)));
        if (in && (i & 15) == 0) a.scales[(size_t)row * a.nblocks + (i >> 4)] = s;
      }
      const float is = 1.0f / s;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= is;
      if (in) *reinterpret_cast<u32x2*>(a.codes + (size_t)row * a.ldc + 8 * i) = to_e4m3(y);
    }
  }
}

constexpr int kNormMaxVpt = 6;

// Lanes and vectors per lane of a row.  Few rows: as many lanes as the row
// feeds (a chain of latencies).  Many: the split with the fewest idle slots,
// and among those the fewest waves, for a row inside one wave needs no LDS.
struct NormPlan {
  int sub, waves, vpt;  // vpt 0: the long kernel
};

inline NormPlan norm_plan(int64_t rows, int nvec, int cus) {
  if (nvec <= 16) return {16, 1, 1};
  if (nvec <= 32) return {32, 1, 1};
  const bool few = rows < 4 * (int64_t)cus;
  NormPlan best{64, 8, 0};
  int64_t best_cost = -1;
  for (int w = 1; w <= 8; w *= 2) {
    const int v = (nvec + 64 * w - 1) / (64 * w);
    if (v > kNormMaxVpt) continue;
    const int64_t cost = few ? v * 1000 + w : (int64_t)w * v * 1000 + w;
    if (best_cost < 0 || cost < best_cost) best = {64, w, v}, best_cost = cost;
  }
  return best;
}

template <typename T, int OUT>
int launch_norm(const NormArgs& a0, hipStream_t s) {
  NormArgs a = a0;
  const NormPlan p = norm_plan(a.rows, a.nvec, device_cu_count());
  if (p.vpt == 0) {
    hipLaunchKernelGGL((rms_norm_long_kernel<T, OUT>), dim3((uint32_t)a.rows), dim3(1024), 0, s, a);
    return launch_status();
  }
  a.waves_per_row = p.waves;
  const int threads = p.waves > 4 ? 64 * p.waves : 256;
  const int lanes = p.sub < 64 ? p.sub : 64 * p.waves;
  const int per = threads / lanes;
  const dim3 grid((uint32_t)((a.rows + per - 1) / per)), block(threads);
#define TP_NORM(SUB, V) hipLaunchKernelGGL((rms_norm_kernel<T, OUT, SUB, V>), grid, block, 0, s, a)
  if (p.sub == 16) TP_NORM(16, 1);
  else if (p.sub == 32) TP_NORM(32, 1);
  else if (p.vpt == 1) TP_NORM(64, 1);
  else if (p.vpt == 2) TP_NORM(64, 2);
  else if (p.vpt == 3) TP_NORM(64, 3);
  else if (p.vpt == 4) TP_NORM(64, 4);
  else if (p.vpt == 5) TP_NORM(64, 5);
  else TP_NORM(64, 6);
#undef TP_NORM
  return launch_status();
}

template <int OUT>
int dispatch_norm(int dtype, const NormArgs& a, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TP_F16) return launch_norm<f16_t, OUT>(a, s);
  if (dtype == TP_BF16) return launch_norm<bf16_t, OUT>(a, s);
  return launch_norm<float, OUT>(a, s);
}

// The checks that both entry points make.
int check_norm(int dtype, int64_t rows, int64_t inner, int64_t d, const void* x, const void* residual,
               const void* weight, const void* h) {
  if (!dtype_ok(dtype)) return TP_ERR_BAD_TYPE;
  if (rows < 0 || rows > 0x7fffffff || inner < 1 || inner > 0x7fffffff || d < 1 || d > (1 << 28)) return TP_ERR_BAD_DIMS;
  if (rows == 0) return TP_OK;
  if (!x || !weight) return TP_ERR_NULL_POINTER;
  const uintptr_t mask = dtype_bytes(dtype) - 1;
  if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)h) & mask) return TP_ERR_MISALIGNED;
  return TP_OK;
}

NormArgs norm_args(int64_t rows, int64_t inner, int64_t d, const void* x, int64_t x_outer, int64_t x_inner,
                   const void* residual, int64_t r_outer, int64_t r_inner, const void* weight, float eps, void* h) {
  NormArgs a{};
  a.x = x, a.residual = residual, a.weight = weight, a.h = h;
  a.x_outer = x_outer, a.x_inner = x_inner, a.r_outer = r_outer, a.r_inner = r_inner;
  a.rows = rows, a.inner = (int)inner, a.d = (int)d, a.nvec = (int)((d + 7) / 8);
  a.nblocks = (int)((d + 127) / 128), a.eps = eps;
  return a;
}

}  // namespace tp

using namespace tp;

extern "C" int tp_rms_norm(int dtype, int64_t rows, int64_t inner, int64_t d, const void* x, int64_t x_outer,
                           int64_t x_inner, const void* residual, int64_t r_outer, int64_t r_inner,
                           const void* weight, float eps, void* y, void* h_out, void* stream) {
  if (const int st = check_norm(dtype, rows, inner, d, x, residual, weight, h_out)) return st;
  if (rows == 0) return TP_OK;
  if (!y) return TP_ERR_NULL_POINTER;
  if ((uintptr_t)y & (dtype_bytes(dtype) - 1)) return TP_ERR_MISALIGNED;
  NormArgs a = norm_args(rows, inner, d, x, x_outer, x_inner, residual, r_outer, r_inner, weight, eps, h_out);
  a.y = y;
  return dispatch_norm<kSame>(dtype, a, stream);
}

extern "C" int tp_rms_norm_fp8(int dtype, int64_t rows, int64_t inner, int64_t d, const void* x, int64_t x_outer,
                               int64_t x_inner, const void* residual, int64_t r_outer, int64_t r_inner,
                               const void* weight, float eps, int block, uint8_t* codes, int64_t ldc,
                               float* scales, void* h_out, void* stream) {
  if (const int st = check_norm(dtype, rows, inner, d, x, residual, weight, h_out)) return st;
  if (block != 0 && block != 128) return TP_ERR_BAD_BLOCK;
  if (ldc < d) return TP_ERR_BAD_DIMS;
  if (rows == 0) return TP_OK;
  if (!codes || !scales) return TP_ERR_NULL_POINTER;
  if ((ldc & 15) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 3)) return TP_ERR_MISALIGNED;
  NormArgs a = norm_args(rows, inner, d, x, x_outer, x_inner, residual, r_outer, r_inner, weight, eps, h_out);
  a.codes = codes, a.ldc = ldc, a.scales = scales;
  return block ? dispatch_norm<kFp8Block>(dtype, a, stream) : dispatch_norm<kFp8Row>(dtype, a, stream);
}
