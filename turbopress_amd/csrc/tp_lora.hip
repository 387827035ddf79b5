// Low-rank adapters of many requests beside a shared projection:
//
//   out[r] = y[r] + scale_i (x[r] A_i^T) B_i^T,  i = adapters[r]
//
// in two launches, h = x A^T, then the rest.  2 rank flops for each element of x
// and y: bound by HBM (x, y and out once, each used adapter's weights once), or by
// latency for few rows.
//
// Rows come in any order of adapters.  A workgroup has 16 (or 64) rows, finds the
// distinct adapters among them, and multiplies all of its rows by each one's
// weights: the matrix instructions' columns are rows, which do not meet, so what
// belongs to another adapter's rows is just not kept.  Of few rows the distinct
// adapters are shared out over further workgroups (`slots`).
//
// The first product is cut along its long sum: parts of fp32, added in order by
// the second launch, which takes h as two numbers of the weights' type, its
// leading bits and what they leave (2^-16 of it are lost in bf16, in fp16, whose
// row is scaled by a power of two to the type's range, 2^-21 of the row's
// largest): one number would lose as much as the output's rounding.
#include "tp_ops_common.h"

#include <algorithm>

namespace tp {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct LoraMma;
template <>
struct LoraMma<f16_t> {
  typedef f16x8 v8;
  __device__ __forceinline__ static f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct LoraMma<bf16_t> {
  typedef bf16x8 v8;
  __device__ __forceinline__ static f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

struct LoraArgs {
  const void *x, *a, *b, *y;
  void* out;
  const int32_t* adapters;
  const float* scales;
  float* h;  // [parts][rows][hr]
  int64_t ldx, ldy, a_adapter, a_row, b_adapter, b_row, rows;
  int k, n, rank, count;
  int parts, slots, hr, steps;  // steps: of 32 columns of x
};

// 8 elements at any alignment, those from `left` on zeros.
template <typename V, typename T>
__device__ __forceinline__ V load_upto(const T* p, int left) {
  V v{};
  if (left >= 8) {
    __builtin_memcpy(&v, p, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) v[e] = p[e];
  }
  return v;
}

// The distinct adapters of the rows whose ids the lanes hold: f(adapter, its rows
// as bits) for every `slots`-th of them, from `slot` on.
template <typename F>
__device__ __forceinline__ void each_adapter(int id, uint64_t pending, int slot, int slots, F f) {
  int turn = 0;
  while (pending) {
    const int who = __builtin_amdgcn_readlane(id, __builtin_ctzll(pending));
    const uint64_t same = __ballot(id == who) & pending;
    pending &= ~same;
    if (turn == slot) f(who, same);
    if (++turn == slots) turn = 0;
  }
}

// h of 16 NT rows and 16 RT ranks over a part of the columns, which W waves share.
template <typename T, int NT, int RT, int W>
__global__ void __launch_bounds__(64 * W) lora_shrink_kernel(const LoraArgs p) {
  typedef typename LoraMma<T>::v8 v8;
  constexpr int ROWS = 16 * NT, U = 4;  // steps whose loads are in flight together
  __shared__ f32x4 sums[W][ROWS][4 * RT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * ROWS;
  const int slot = blockIdx.z % p.slots, rank0 = blockIdx.z / p.slots * 16 * RT;
  const int id = lane < ROWS && row0 + lane < p.rows ? p.adapters[row0 + lane] : -1;
  const int from = (int)((int64_t)p.steps * blockIdx.y / p.parts), to = (int)((int64_t)p.steps * (blockIdx.y + 1) / p.parts);
  const int s0 = from + (to - from) * wave / W, s1 = from + (to - from) * (wave + 1) / W;
  const T* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = static_cast<const T*>(p.x) + min(row0 + 16 * t + lr, p.rows - 1) * p.ldx + 8 * lg;

  each_adapter(id, __ballot(id >= 0 && id < p.count), slot, p.slots, [&](int who, uint64_t same) __attribute__((always_inline)) {
    const T* a[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
      a[r] = static_cast<const T*>(p.a) + who * p.a_adapter + min(rank0 + 16 * r + lr, p.rank - 1) * p.a_row + 8 * lg;
    f32x4 acc[NT][RT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[t][r] = f32x4{0, 0, 0, 0};
    for (int s = s0; s < s1; s += U) {
      v8 xv[U][NT], av[U][RT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = 32 * (s + u);
        if (s + u < s1 && c + 32 <= p.k) {
#pragma unroll
          for (int t = 0; t < NT; ++t) __builtin_memcpy(&xv[u][t], x[t] + c, 16);
#pragma unroll
          for (int r = 0; r < RT; ++r) __builtin_memcpy(&av[u][r], a[r] + c, 16);
        } else {
          const int left = s + u < s1 ? p.k - c - 8 * lg : 0;
#pragma unroll
          for (int t = 0; t < NT; ++t) xv[u][t] = load_upto<v8>(x[t] + c, left);
#pragma unroll
          for (int r = 0; r < RT; ++r) av[u][r] = load_upto<v8>(a[r] + c, left);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < RT; ++r) acc[t][r] = LoraMma<T>::mul(av[u][r], xv[u][t], acc[t][r]);
    }
    // lane: row 16 t + lr, ranks 16 r + 4 lg .. + 3
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) sums[wave][16 * t + lr][4 * r + lg] = acc[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * 4 * RT; i += 64 * W) {
      const int row = i / (4 * RT), c = i - row * (4 * RT);
      if (same >> row & 1) {
        f32x4 sum = sums[0][row][c];
#pragma unroll
        for (int w = 1; w < W; ++w) sum += sums[w][row][c];
        *reinterpret_cast<f32x4*>(p.h + (blockIdx.y * p.rows + row0 + row) * p.hr + rank0 + 4 * c) = sum;
      }
    }
    __syncthreads();
  });
}

// The outputs of 16 NT rows and 256 columns.  LDS: h as two operands [step of 32
// ranks][16 rows][lane], then each row's power of two.
template <typename T, int NT>
__global__ void __launch_bounds__(256) lora_expand_kernel(const LoraArgs p) {
  typedef typename LoraMma<T>::v8 v8;
  constexpr int ROWS = 16 * NT;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * ROWS;
  const int slot = blockIdx.z, steps = (p.rank + 31) / 32;
  v8* lead = reinterpret_cast<v8*>(lds);
  v8* rest = lead + steps * NT * 64;
  int* power = reinterpret_cast<int*>(rest + steps * NT * 64);
  const int id = lane < ROWS && row0 + lane < p.rows ? p.adapters[row0 + lane] : -1;
  const uint64_t valid = __ballot(id >= 0 && id < p.count);
  const uint64_t here = __ballot(lane < ROWS && row0 + lane < p.rows);
  // this workgroup's rows
  uint64_t mine = 0;
  each_adapter(id, valid, slot, p.slots, [&](int, uint64_t same) __attribute__((always_inline)) { mine |= same; });
  const uint64_t plain = slot == 0 ? here & ~valid : 0;  // rows without an adapter
  if (!(mine | plain)) return;

  // their h, 8 threads a row, 8 ranks at a time
  for (int row = threadIdx.x / 8; row < ROWS; row += 32) {
    if (!(mine >> row & 1)) continue;
    const int l8 = threadIdx.x & 7;
    const int who = p.adapters[row0 + row];
    const float scale = p.scales ? p.scales[who] : 1.0f;
    const float* h = p.h + (row0 + row) * p.hr;
    float most = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {  // (fp16: its largest first)
      int up = 0;
      if constexpr (__is_same(T, f16_t)) {
        if (pass == 1) {
#pragma unroll
          for (int o = 1; o < 8; o *= 2) most = fmaxf(most, __shfl_xor(most, o));
          if (most > 0.0f && most < INFINITY) up = 15 - __builtin_amdgcn_frexp_expf(most);
          if (l8 == 0) power[row] = -up;
        }
      } else if (pass == 0) {
        continue;
      }
      for (int c = l8; c < 4 * steps; c += 8) {
        f32x4 v[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
        if (8 * c < p.rank) {
          for (int part = 0; part < p.parts; ++part) {
            const f32x4* q = reinterpret_cast<const f32x4*>(h + part * p.rows * p.hr + 8 * c);
            v[0] += q[0];
            v[1] += q[1];
          }
        }
        v8 a, b;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float f = 8 * c + e < p.rank ? v[e / 4][e % 4] * scale : 0.0f;
          if constexpr (__is_same(T, f16_t)) {
            if (pass == 0) most = fmaxf(most, fabsf(f));
            f = __builtin_ldexpf(f, up);
          }
          a[e] = (T)f;
          const float r = f - (float)a[e];
          b[e] = (T)(r - r == 0.0f ? r : 0.0f);  // (of infinity and NaN nothing is left)
        }
        if (pass == 1) {
          const int at = ((c / 4 * NT + row / 16) * 4 + c % 4) * 16 + row % 16;
          lead[at] = a, rest[at] = b;
        }
      }
    }
  }
  __syncthreads();

  // A lane has 16 columns of a row: tile t's row 4 g + e of the matrix instruction
  // is column 16 g + 4 t + e.
  const int column0 = blockIdx.y * 256 + wave * 64, column = column0 + 16 * lg;
  if (column0 >= p.n) return;
  auto put = [&](int t, uint64_t rows, const f32x4 (&acc)[4], int up) __attribute__((always_inline)) {
    const int row = 16 * t + lr;
    if (!(rows >> row & 1)) return;
    const T* y = static_cast<const T*>(p.y) + (row0 + row) * p.ldy + column;
    T* out = static_cast<T*>(p.out) + (row0 + row) * p.n + column;
    struct {
      T v[16];
    } r;
    if (column + 16 <= p.n) {
      __builtin_memcpy(&r, y, sizeof(r));
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) r.v[e] = column + e < p.n ? y[e] : (T)0.0f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float f = acc[e / 4][e % 4];
      if constexpr (__is_same(T, f16_t)) f = __builtin_ldexpf(f, up);
      r.v[e] = (T)((float)r.v[e] + f);
    }
    if (column + 16 <= p.n) {
      __builtin_memcpy(out, &r, sizeof(r));
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (column + e < p.n) out[e] = r.v[e];
    }
  };
  each_adapter(id, valid, slot, p.slots, [&](int who, uint64_t same) __attribute__((always_inline)) {
    const T* b[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
      b[t] = static_cast<const T*>(p.b) + who * p.b_adapter + min(column0 + 16 * (lr >> 2) + 4 * t + (lr & 3), p.n - 1) * p.b_row + 8 * lg;
    f32x4 acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[t][c] = f32x4{0, 0, 0, 0};
    for (int s = 0; s < steps; ++s) {
      v8 w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = load_upto<v8>(b[c] + 32 * s, p.rank - 32 * s - 8 * lg);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const v8 h0 = lead[(s * NT + t) * 64 + lane], h1 = rest[(s * NT + t) * 64 + lane];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          acc[t][c] = LoraMma<T>::mul(w[c], h0, acc[t][c]);
          acc[t][c] = LoraMma<T>::mul(w[c], h1, acc[t][c]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) put(t, same, acc[t], __is_same(T, f16_t) ? power[16 * t + lr] : 0);
  });
  const f32x4 zero[4] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
  if (plain) {
#pragma unroll
    for (int t = 0; t < NT; ++t) put(t, plain, zero, 0);
  }
}

struct LoraPlan {
  int tiles, parts, slots, hr, steps;  // tiles: of 16 rows of a workgroup
};

inline LoraPlan lora_plan(int64_t rows, int64_t k, int64_t rank) {
  LoraPlan q;
  q.tiles = rows > 256 ? 4 : 1;
  q.slots = q.tiles == 1 ? 16 : 1;
  q.hr = (int)(rank + 63) / 64 * 64;
  q.steps = (int)(k + 31) / 32;
  const int64_t groups = (rows + 16 * q.tiles - 1) / (16 * q.tiles), waves = q.tiles == 1 ? 4 : 8;
  int64_t parts = (q.steps + 5 * waves - 1) / (5 * waves);
  if (q.tiles > 1) parts = std::min(parts, std::max((int64_t)1, (256 + groups - 1) / groups));
  q.parts = (int)std::min(parts, (int64_t)16);
  return q;
}

template <typename T, int NT, int RT, int W>
void launch_shrink(const LoraArgs& p, hipStream_t s) {
  const dim3 grid((uint32_t)((p.rows + 16 * NT - 1) / (16 * NT)), p.parts, p.slots * ((p.rank + 16 * RT - 1) / (16 * RT)));
  hipLaunchKernelGGL((lora_shrink_kernel<T, NT, RT, W>), grid, dim3(64 * W), 0, s, p);
}

template <typename T, int NT, int W>
int launch_lora(const LoraArgs& p, hipStream_t s) {
  if (p.count > 0) {
    if (p.rank <= 16) launch_shrink<T, NT, 1, W>(p, s);
    else if (p.rank <= 32) launch_shrink<T, NT, 2, W>(p, s);
    else launch_shrink<T, NT, 4, W>(p, s);
  }
  const int steps = (p.rank + 31) / 32, bytes = steps * NT * 2048 + NT * 64;
  allow_dynamic_lds(reinterpret_cast<const void*>(lora_expand_kernel<T, NT>), 0);
  const dim3 grid((uint32_t)((p.rows + 16 * NT - 1) / (16 * NT)), (p.n + 255) / 256, p.slots);
  hipLaunchKernelGGL((lora_expand_kernel<T, NT>), grid, dim3(256), bytes, s, p);
  return launch_status();
}

inline bool lora_sizes_ok(int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count) {
  return rows >= 0 && rows <= (1 << 24) && k >= 1 && k <= (1 << 20) && n >= 1 && n <= (1 << 20) && rank >= 1 && rank <= 256 &&
         count >= 0 && count <= (1 << 20) && grid_fits((rows + 63) / 64 * ((n + 255) / 256), 256);
}

}  // namespace tp

using namespace tp;

extern "C" int64_t tp_lora_workspace_bytes(int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count) {
  if (!lora_sizes_ok(rows, k, n, rank, count)) return -1;
  const LoraPlan q = lora_plan(rows, k, rank);
  return count ? rows * q.parts * q.hr * (int64_t)sizeof(float) : 0;
}

extern "C" int tp_lora_add(int dtype, int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count, const void* x,
                           int64_t ldx, const void* a, int64_t a_adapter, int64_t a_row, const void* b,
                           int64_t b_adapter, int64_t b_row, const int32_t* adapters, const float* scales,
                           const void* y, int64_t ldy, void* out, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  if (dtype != TP_F16 && dtype != TP_BF16) return TP_ERR_BAD_TYPE;
  if (!lora_sizes_ok(rows, k, n, rank, count) || ldx < 0 || ldy < 0) return TP_ERR_BAD_DIMS;
  if (rows == 0) return TP_OK;
  if (!x || !y || !out || !adapters || (count && (!a || !b))) return TP_ERR_NULL_POINTER;
  if ((((uintptr_t)x | (uintptr_t)a | (uintptr_t)b | (uintptr_t)y | (uintptr_t)out) & 1) || (((uintptr_t)adapters | (uintptr_t)scales) & 3))
    return TP_ERR_MISALIGNED;
  const int64_t need = tp_lora_workspace_bytes(rows, k, n, rank, count);
  if (need && (!workspace || workspace_bytes < need)) return TP_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return TP_ERR_MISALIGNED;
  const LoraPlan q = lora_plan(rows, k, rank);
  LoraArgs p{};
  p.x = x, p.a = a, p.b = b, p.y = y, p.out = out, p.adapters = adapters, p.scales = scales, p.h = static_cast<float*>(workspace);
  p.ldx = ldx, p.ldy = ldy, p.a_adapter = a_adapter, p.a_row = a_row, p.b_adapter = b_adapter, p.b_row = b_row;
  p.rows = rows, p.k = (int)k, p.n = (int)n, p.rank = (int)rank, p.count = (int)count;
  p.parts = q.parts, p.slots = q.slots, p.hr = q.hr, p.steps = q.steps;
  hipStream_t s = (hipStream_t)stream;
  if (q.tiles == 1) return dtype == TP_F16 ? launch_lora<f16_t, 1, 4>(p, s) : launch_lora<bf16_t, 1, 4>(p, s);
  return dtype == TP_F16 ? launch_lora<f16_t, 4, 8>(p, s) : launch_lora<bf16_t, 4, 8>(p, s);
}
