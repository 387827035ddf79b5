// Root-mean-square norm of rows, with the residual's addition, its output in
// the input's type or in 8-bit floating point with scales:
//
//   h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight
//   scale = max(max |y| / 448, 2^-126),  code = e4m3(y / scale)
//
// One pass: a row's x and residual stay in registers between its sum of squares
// and its output, so they are read once and h, y (or codes) written once; the
// weight comes from L2.  4 flops per element (a wave's vector instructions for 64
// of them: 16 of fp16 rows off their words, 29 with a residual and e4m3 output, for
// conversions, maxima and quotients): many rows are bound by HBM, a few by the latency of load, reduction
// and store.  8192 x 9728 fp16 60 us = 5.3 TB/s (a copy reaches 5.2); 8191 x 9727
// 70, half of its rows off their words; 2048 x 2560 with a residual and e4m3
// output 10.2 (scales per row 10.0), of which the instructions' issue alone is 3.9;
// 1 x 2560 3.0.
#include "tp_ops_common.h"

#include <algorithm>
#include <type_traits>

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
  int large;  // the inputs are past the caches' size
  int odd;    // rows of 2-byte elements that do not all begin on words
  float eps;
};

enum NormOut { kSame = 0, kFp8Block = 1, kFp8Row = 2 };

constexpr float kE4m3Max = 448.0f;
constexpr float kLeastScale = 0x1p-126f;

// Elements [8 i, 8 i + 8) of a row of d, zeros past its end.
template <bool ONCE = false, typename T>
__device__ __forceinline__ Vec<T> load_row8(const T* row, int i, int d) {
  if (8 * i + 8 <= d) return ONCE ? load8_once(row + 8 * i) : load8(row + 8 * i);
  Vec<T> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = 8 * i + e < d ? row[8 * i + e] : (T)0.0f;
  return r;
}

template <typename T>
__device__ __forceinline__ void store_row8(T* row, int i, int d, const Vec<T>& r) {
  if (8 * i + 8 <= d) {
    store8_once(row + 8 * i, r);
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

// y / s as a division rounds it (codes at ties depend on its last bit), with one
// reciprocal for all that share s: the product with 1 / s is off by a unit or so,
// and its remainder q s - y, exact in an FMA, sets it right (Markstein's
// method; zeros keep their signs).  A division's own steps, per element, are
// about ten instructions; these are three.
struct Divisor {
  float s, inv;
  __device__ __forceinline__ explicit Divisor(float scale) : s(scale), inv(1.0f / scale) {
    if (inv == 0.0f) s = 0.0f;  // (an infinite scale: zeros, as finite / infinite, and NaN of infinite y)
  }
  __device__ __forceinline__ float of(float y) const {
    const float q = y * inv;
    return fmaf(-fmaf(q, s, -y), inv, q);
  }
};

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
// vectors of 8 elements per lane, one row each.  What stays in registers across
// the reduction is x and the residual as they were loaded; h is formed again
// behind it.  (8192 x 9728 fp16: with h kept in fp32 and the weight beside it
// 100 us, and 102 with workgroups that go on to further rows, the next one's
// loads in flight: either leaves fewer waves to a CU, and the loads of some
// waves have to run under the reductions and stores of others.)
template <typename T, int OUT, bool RES, int SUB, int VPT>
__global__ void __launch_bounds__(512) rms_norm_kernel(const NormArgs a) {
  __shared__ float slots[32];
  const int wpr = SUB < 64 ? 1 : a.waves_per_row;
  const int lanes = SUB < 64 ? SUB : 64 * wpr;  // that hold one row
  const int i0 = (int)threadIdx.x & (lanes - 1);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / lanes) + (int)threadIdx.x / lanes;
  const bool live = row < a.rows;
  const int64_t rrow = live ? row : a.rows - 1;  // (idle lanes follow a row along, for the barriers)
  const T* x = static_cast<const T*>(a.x) + row_offset(rrow, a.inner, a.x_outer, a.x_inner);
  const T* res = RES ? static_cast<const T*>(a.residual) + row_offset(rrow, a.inner, a.r_outer, a.r_inner) : nullptr;
  const T* weight = static_cast<const T*>(a.weight);
  const int last = a.nvec - 1;  // (lanes past the row load its last vector, and add nothing)

  Vec<T> xv[VPT], rv[RES ? VPT : 1];
  auto load = [&](auto once) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) xv[j] = load_row8<decltype(once)::value>(x, min(i0 + j * lanes, last), a.d);
    if constexpr (RES) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) rv[j] = load_row8<decltype(once)::value>(res, min(i0 + j * lanes, last), a.d);
    }
  };
  // The word behind a vector is the next lane's first (loaded by every lane, 8191
  // x 9727 fp16 took 79 us, no less than unaligned), but for a wave's or a row's
  // last lane.  All vectors are loaded, then moved.
  auto load_odd = [&](auto once) __attribute__((always_inline)) {
    Unaligned<4> xu[VPT], ru[RES ? VPT : 1];
    auto get = [&](Unaligned<4>& u, const T* r, int i) __attribute__((always_inline)) {
      if (8 * i + 8 <= a.d) u.load<decltype(once)::value>(r + 8 * i, i == last || (i0 & (SUB - 1)) == SUB - 1);
      else u.load_first(r + 8 * i, (a.d - 8 * i) * (int)sizeof(T));
    };
    auto moved = [&](Vec<T>& v, Unaligned<4>& u, const T* r, int i) __attribute__((always_inline)) {
      const uint32_t s = (uint32_t)(uintptr_t)r & 3, behind = from_next_lane(u.at[0][0]);
      if (i != last && (i0 & (SUB - 1)) != SUB - 1) u.next = behind;
      const u32x4 w = {u.word(0, s), u.word(1, s), u.word(2, s), u.word(3, s)};
      __builtin_memcpy(&v, &w, 16);
    };
#pragma unroll
    for (int j = 0; j < VPT; ++j) get(xu[j], x, min(i0 + j * lanes, last));
    if constexpr (RES) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) get(ru[j], res, min(i0 + j * lanes, last));
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      moved(xv[j], xu[j], x, min(i0 + j * lanes, last));
      if constexpr (RES) moved(rv[j], ru[j], res, min(i0 + j * lanes, last));
    }
  };
  if (sizeof(T) == 2 && a.odd) {
    if constexpr (sizeof(T) == 2) {
      if (a.large) load_odd(std::true_type{});
      else load_odd(std::false_type{});
    }
  } else if (a.large) {
    load(std::true_type{});
  } else {
    load(std::false_type{});
  }
  auto sum8 = [&](int j, float* h) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = (float)xv[j].v[e];
      if constexpr (RES) h[e] += (float)rv[j].v[e];
    }
  };
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    float h[8], part = 0.0f;
    sum8(j, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) part = fmaf(h[e], h[e], part);
    sum += i0 + j * lanes <= last ? part : 0.0f;
    if (RES && a.h && live && i0 + j * lanes <= last) {
      Vec<T> o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = (T)h[e];
      store_row8(static_cast<T*>(a.h) + (size_t)row * a.d, i0 + j * lanes, a.d, o);
    }
  }
  if (!RES && a.h && live) {  // (without a residual h is x)
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (i0 + j * lanes <= last) store_row8(static_cast<T*>(a.h) + (size_t)row * a.d, i0 + j * lanes, a.d, xv[j]);
  }
  Vec<T> wv[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) wv[j] = load_row8(weight, min(i0 + j * lanes, last), a.d);
  sum = reduce_row<AddOp, SUB>(sum, wpr, slots);
  const float inv = 1.0f / sqrtf(sum / (float)a.d + a.eps);
  auto norm8 = [&](int j, float* y) __attribute__((always_inline)) {
    sum8(j, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * (float)wv[j].v[e];
  };

  if constexpr (OUT == kSame) {
    T* yr = static_cast<T*>(a.y) + (size_t)row * a.d;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (live && i0 + j * lanes <= last) {
        float y[8];
        norm8(j, y);
        Vec<T> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = (T)y[e];
        store_row8(yr, i0 + j * lanes, a.d, o);
      }
  } else {
    float s_row = 0.0f;
    if constexpr (OUT == kFp8Row) {
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {  // (the last vector again, in lanes past it, changes no maximum)
        float y[8];
        norm8(j, y);
        m = MaxNanOp::of(m, max_abs8(y));
      }
      s_row = scale_of(reduce_row<MaxNanOp, SUB>(m, wpr, slots + 16));
      if (live && i0 == 0) a.scales[row] = s_row;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = i0 + j * lanes;
      float y[8], s = s_row;
      norm8(j, y);
      if constexpr (OUT == kFp8Block) {  // 16 lanes hold a block of 128 (of its vectors, lanes past the row the last)
        s = scale_of(reduce16<MaxNanOp>(max_abs8(y)));
        if (live && i <= last && (i & 15) == 0) a.scales[(size_t)row * a.nblocks + (i >> 4)] = s;
      }
      const Divisor by(s);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = by.of(y[e]);
      if (live && i <= last) __builtin_nontemporal_store(to_e4m3(y), reinterpret_cast<u32x2*>(a.codes + (size_t)row * a.ldc + 8 * i));
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
      const Divisor by(s);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = by.of(y[e]);
      if (in) *reinterpret_cast<u32x2*>(a.codes + (size_t)row * a.ldc + 8 * i) = to_e4m3(y);
    }
  }
}

constexpr int kNormMaxVpt = 6;

// Lanes and vectors per lane of a row.  Few rows: as many lanes as the row
// feeds (a chain of latencies).  Many: the split with the fewest idle slots,
// and among those the fewest waves, for a row inside one wave needs no LDS.
// Few are up to 4 per CU, 2 with a scale per row (whose maximum is a second chain
// through LDS), 8 of fp32 in and out.  With a residual, us, the split of many rows
// / of few:
//           fp16                            bf16 -> e4m3 per 128
//   d       1 row    512      1024     2048      512      1024     2048
//   1024    3.1/2.7  3.6/3.2  3.9/3.6  4.5/4.5   4.1/3.5  4.2/3.8  4.9/4.9
//   2560    4.6/3.0  5.5/4.4  6.2/6.0  8.4/9.3   6.5/4.8  7.2/6.7  9.8/10.8
//   4096    4.3/3.2  5.3/4.6  7.4/7.2  12/12.2   6.3/5.0  8.7/8.2  13.2/13.5
//   9728    5.2/4.2  8.5/7.8  14/13.4  27/25.3   9.9/9.4  16/16.3  27.7/27.8
//           bf16 -> e4m3 per row            fp32
//   1024    3.4/3.2  4.0/3.7  4.2/4.1  4.9/5.1   3.6/3.4  4.3/4.2  7.6/7.6
//   2560    5.0/3.8  6.0/5.4  6.8/7.6  9.0/12.1  6.3/5.1  8.6/8.5  19/16.0
//   4096    4.9/3.8  6.0/5.5  8.2/8.8  13/14.3   7.5/7.3  15/13.2  25.7/25.2
//   9728    5.8/5.0  9.5/9.3  14.6/16  27/27.2   17/15.6  31/28.9  65/66.7
struct NormPlan {
  int sub, waves, vpt;  // vpt 0: the long kernel
};

inline NormPlan norm_plan(int64_t rows, int nvec, int64_t few_rows) {
  if (nvec <= 16) return {16, 1, 1};
  if (nvec <= 32) return {32, 1, 1};
  const bool few = rows <= few_rows;
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
  // Loads past the caches from 128 MB of inputs, half of what the memory side
  // caches: 8192 x 9728 fp16 60 us against 67, 16384 x
  // 2560 with a residual 65 against 66; what the step before has just written is
  // better read from there: 16384 x 1024 with a residual 25.8 against 21.1, 2048 x
  // 2560 13.5 against 9.0, 4096 x 9728 without 33 against 31.
  a.large = a.rows * a.d * (int64_t)sizeof(T) * (a.residual ? 2 : 1) >= (128 << 20);
  const int64_t at = (int64_t)(uintptr_t)a.x | (int64_t)(uintptr_t)a.residual |
                     ((a.x_outer | a.x_inner | a.r_outer | a.r_inner) * (int64_t)sizeof(T));
  a.odd = (at & 3) != 0;
  constexpr int64_t kFewPerCu = OUT == kFp8Row ? 2 : OUT == kSame && sizeof(T) == 4 ? 8 : 4;
  const NormPlan p = norm_plan(a.rows, a.nvec, kFewPerCu * device_cu_count());
  if (p.vpt == 0) {
    if (!grid_fits(a.rows, 1024)) return TP_ERR_BAD_DIMS;
    hipLaunchKernelGGL((rms_norm_long_kernel<T, OUT>), dim3((uint32_t)a.rows), dim3(1024), 0, s, a);
    return launch_status();
  }
  a.waves_per_row = p.waves;
  const int threads = p.waves > 4 ? 64 * p.waves : 256;
  const int lanes = p.sub < 64 ? p.sub : 64 * p.waves;
  const int per = threads / lanes;
  if (!grid_fits((a.rows + per - 1) / per, threads)) return TP_ERR_BAD_DIMS;
  const dim3 grid((uint32_t)((a.rows + per - 1) / per)), block(threads);
#define TP_NORM(SUB, V)                                                                              \
  do {                                                                                               \
    if (a.residual) hipLaunchKernelGGL((rms_norm_kernel<T, OUT, true, SUB, V>), grid, block, 0, s, a); \
    else hipLaunchKernelGGL((rms_norm_kernel<T, OUT, false, SUB, V>), grid, block, 0, s, a);           \
  } while (0)
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
