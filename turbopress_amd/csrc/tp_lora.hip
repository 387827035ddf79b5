// Low-rank adapters of many requests beside a shared projection:
//
//   out[r] = y[r] + scale_i (x[r] A_i^T) B_i^T,  i = adapters[r]
//
// in two launches, h = x A^T, then the rest (three where the first product's long
// sum is cut).  2 rank flops for each element of x
// and y: bound by HBM (x, y and out once, each used adapter's weights once), or by
// latency for few rows.
//
// Rows come in any order of adapters.  A workgroup has 16 (or 64) rows, finds the
// distinct adapters among them, and multiplies all of its rows by each one's
// weights: the matrix instructions' columns are rows, which do not meet, so what
// belongs to another adapter's rows is just not kept.  Of few rows the distinct
// adapters are shared out over further workgroups (`slots`).
//
// h is left in the order of the second product's operands, as two numbers of the
// weights' type, its leading bits and what they leave (2^-16 of it are lost in
// bf16, in fp16, where 32 ranks of a row are scaled by a power of two to the type's
// range, 2^-21 of their largest): one number would lose as much as the output's
// rounding.
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
  float* parts_h;     // [parts][rows][hr], where there are several
  void *lead, *rest;  // h's two numbers: [16 rows][step of 32 ranks][lane] operands
  int* power;         // fp16: [rows][step], the power of two of h
  int64_t ldx, ldy, a_adapter, a_row, b_adapter, b_row, rows;
  int k, n, rank, count;
  int parts, slots, hr, lines, steps;  // lines: of 64 columns of a row of x
};

// 8 elements at any alignment.
template <typename V, typename T>
__device__ __forceinline__ V load_eight(const T* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(v));
  return v;
}
// Those from `left` on zeros; the row's last element, at left - 1, may be read in
// their place (left may be 0 and less: no branch, the loads are in flight together).
template <typename V, typename T>
__device__ __forceinline__ V load_upto(const T* p, int left) {
  V v;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const T x = p[min(e, left - 1)];
    v[e] = e < left ? x : (T)0.0f;
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

// 8 ranks from 8 c on of a row's h (its sums v, unscaled), by four lanes a step of
// 32 (aligned in their wave, all of them active).
template <typename T>
__device__ __forceinline__ void leave_h(const LoraArgs& p, int64_t row, int c, f32x4 (&v)[2], float scale) {
  typedef typename LoraMma<T>::v8 v8;
  float most = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float f = 8 * c + e < p.rank ? v[e / 4][e % 4] * scale : 0.0f;
    v[e / 4][e % 4] = f;
    most = fmaxf(most, fabsf(f));
  }
  int up = 0;
  if constexpr (__is_same(T, f16_t)) {
    most = fmaxf(most, __shfl_xor(most, 1));
    most = fmaxf(most, __shfl_xor(most, 2));
    if (most > 0.0f && most < INFINITY) up = 15 - __builtin_amdgcn_frexp_expf(most);
    if (c % 4 == 0 && c / 4 < p.steps) p.power[row * p.steps + c / 4] = -up;
  }
  if (c / 4 >= p.steps) return;
  v8 a, b;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float f = v[e / 4][e % 4];
    if constexpr (__is_same(T, f16_t)) f = __builtin_ldexpf(f, up);
    a[e] = (T)f;
    const float r = f - (float)a[e];
    b[e] = (T)(r - r == 0.0f ? r : 0.0f);  // (of infinity and NaN nothing is left)
  }
  const int64_t to = ((row / 16 * p.steps + c / 4) * 4 + c % 4) * 16 + row % 16;
  static_cast<v8*>(p.lead)[to] = a, static_cast<v8*>(p.rest)[to] = b;
}

// Columns of x that a wave takes at once: a row's are a line of 128 bytes.
constexpr int kLine = 64;

// h of 16 NT rows and 16 RT ranks over a part of the columns, which W waves share.
// A wave loads whole lines, 8 lanes each (operands straight from memory would be 64
// accesses of 16 bytes: 2047 x 9728 of rank 64 30 us), and turns them into operands
// in LDS of its own: piece c of row r lies at c ^ (r & 7), so that 16 rows' pieces
// are on distinct banks.  Bound by the waits for lines: 2047 x 9728 of rank 64 18.7 us =
// 2.1 TB/s, matrix units busy for a seventh of it.
template <typename T, int NT, int RT, int W>
__global__ void __launch_bounds__(64 * W) lora_shrink_kernel(const LoraArgs p) {
  typedef typename LoraMma<T>::v8 v8;
  constexpr int ROWS = 16 * NT, LINES = 16 * (NT + RT);  // lines: of x's rows, then of A's
  constexpr int kSums = ROWS * (4 * RT + 1);             // (a piece more a row: 16 rows' pieces on distinct banks)
  constexpr int kWave = kSums > LINES * 8 ? kSums : LINES * 8;
  constexpr int PIECES = RT < 2 ? 4 : 2 * RT;  // of 8 ranks that a row leaves
  static_assert(ROWS * PIECES <= 64 * W, "a thread has one piece at most");
  __shared__ f32x4 lds[W][kWave];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * ROWS;
  const int slot = blockIdx.z % p.slots, rank0 = blockIdx.z / p.slots * 16 * RT;
  const int id = lane < ROWS && row0 + lane < p.rows ? p.adapters[row0 + lane] : -1;
  const int from = (int)((int64_t)p.lines * blockIdx.y / p.parts), to = (int)((int64_t)p.lines * (blockIdx.y + 1) / p.parts);
  const int s0 = from + (to - from) * wave / W, s1 = from + (to - from) * (wave + 1) / W;
  const int whole = min(s1, p.k / kLine);  // lines of 64 columns up to here
  const int at = lane >> 3, piece = lane & 7;  // of what the lane loads
  v8* staged = reinterpret_cast<v8*>(lds[wave]);
  const int own_row = threadIdx.x / PIECES, own_piece = threadIdx.x % PIECES;  // of h
  const int own_id = __shfl(id, own_row < ROWS ? own_row : 0);
  const T* x = static_cast<const T*>(p.x) + row0 * p.ldx;

  each_adapter(id, __ballot(id >= 0 && id < p.count), slot, p.slots, [&](int who, uint64_t same) __attribute__((always_inline)) {
    const T* a = static_cast<const T*>(p.a) + who * p.a_adapter + rank0 * p.a_row;
    // the lane's eight columns of line 8 i + at (rows are at most 2^24 apart: 32 bits)
    auto line = [&](int i, int s) __attribute__((always_inline)) {
      const int l = 8 * i + at;
      const int to = i < 2 * NT ? l * (int)p.ldx : min(l - ROWS, p.rank - 1 - rank0) * (int)p.a_row;
      return (i < 2 * NT ? x : a) + kLine * s + (to + 8 * piece);
    };
    // (rows of other adapters are not read: what lies in LDS there is not kept)
    auto wanted = [&](int i) __attribute__((always_inline)) { return i >= 2 * NT || (same >> (8 * i + at) & 1); };
    f32x4 acc[NT][RT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[t][r] = f32x4{0, 0, 0, 0};
    auto multiply = [&]() __attribute__((always_inline)) {
      wave_lds_fence();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        v8 xv[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) xv[t] = staged[(16 * t + lr) * 8 + ((4 * u + lg) ^ (lr & 7))];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const v8 w = staged[(ROWS + 16 * r + lr) * 8 + ((4 * u + lg) ^ (lr & 7))];
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][r] = LoraMma<T>::mul(w, xv[t], acc[t][r]);
        }
      }
      wave_lds_fence();
    };
    v8 v[2 * (NT + RT)];
    auto load = [&](int s) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2 * (NT + RT); ++i)
        if (wanted(i)) v[i] = load_eight<v8>(line(i, s));
    };
    if (s0 < whole) load(s0);
    for (int s = s0; s < whole; ++s) {
#pragma unroll
      for (int i = 0; i < 2 * (NT + RT); ++i) staged[(8 * i + at) * 8 + (piece ^ at)] = v[i];
      if (s + 1 < whole) load(s + 1);
      multiply();
    }
    if (whole < s1) {  // the row's end
#pragma unroll 1
      for (int i = 0; i < 2 * (NT + RT); ++i)
        if (wanted(i))
          staged[(8 * i + at) * 8 + (piece ^ at)] = load_upto<v8>(line(i, whole), p.k - kLine * whole - 8 * piece);
      multiply();
    }
    // lane: row 16 t + lr, ranks 16 r + 4 lg .. + 3
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < RT; ++r) lds[wave][(16 * t + lr) * (4 * RT + 1) + 4 * r + lg] = acc[t][r];
    __syncthreads();
    if (own_row < ROWS && same >> own_row & 1) {
      f32x4 sum[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
      if (own_piece < 2 * RT) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          sum[c] = lds[0][own_row * (4 * RT + 1) + 2 * own_piece + c];
#pragma unroll
          for (int w = 1; w < W; ++w) sum[c] += lds[w][own_row * (4 * RT + 1) + 2 * own_piece + c];
        }
      }
      if (p.parts == 1) {
        leave_h<T>(p, row0 + own_row, rank0 / 8 + own_piece, sum, p.scales ? p.scales[own_id] : 1.0f);
      } else if (own_piece < 2 * RT) {
        f32x4* q = reinterpret_cast<f32x4*>(p.parts_h + (blockIdx.y * p.rows + row0 + own_row) * p.hr + rank0 + 8 * own_piece);
        q[0] = sum[0], q[1] = sum[1];
      }
    }
    __syncthreads();
  });
}

// The parts' sums, added in order: a thread per row and 8 ranks.
template <typename T>
__global__ void __launch_bounds__(256) lora_join_kernel(const LoraArgs p) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / (4 * p.steps);
  const int c = (int)(at - row * (4 * p.steps));
  if (row >= p.rows) return;
  const int who = p.adapters[row];
  if (who < 0 || who >= p.count) return;
  f32x4 sum[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
  // (h has room for whole pieces of 16 ranks: past those nothing is read)
  const float* h = p.parts_h + row * p.hr + 8 * min(c, (p.rank - 1) / 8);
  for (int part = 0; part < p.parts; part += 4) {
    f32x4 q[4][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const f32x4* from = reinterpret_cast<const f32x4*>(h + min(part + u, p.parts - 1) * p.rows * p.hr);
      q[u][0] = from[0], q[u][1] = from[1];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (part + u < p.parts) sum[0] += q[u][0], sum[1] += q[u][1];
  }
  leave_h<T>(p, row, c, sum, p.scales ? p.scales[who] : 1.0f);
}

// The outputs of 16 NT rows and 256 columns (64 rows of 32 adapters of rank 64, 2560 ->
// 9728 bf16: 15.5 us, of which 45 MB of weights take 7; 2047 rows, 9728 -> 2560 fp16 12.6,
// y in and out 4.1).  PLAIN: a rank that is a
// multiple of 8 and 64 columns and more, of which the last wave takes the last 64.
// Loads that need no other's result are issued together: the ids, then y, h and the
// first weights; the next step's while one is multiplied.
template <typename T, int NT, bool PLAIN>
__global__ void __launch_bounds__(256) lora_expand_kernel(const LoraArgs p) {
  typedef typename LoraMma<T>::v8 v8;
  constexpr int ROWS = 16 * NT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * ROWS;
  const int slot = blockIdx.z;
  // A lane has 16 columns of a row: tile t's row 4 g + e of the matrix instruction
  // is column 16 g + 4 t + e.
  if (blockIdx.y * 256 + wave * 64 >= (uint32_t)p.n) return;
  const int column0 = PLAIN ? min((int)blockIdx.y * 256 + wave * 64, p.n - 64) : (int)blockIdx.y * 256 + wave * 64;
  const int column = column0 + 16 * lg;
  const int id = lane < ROWS && row0 + lane < p.rows ? p.adapters[row0 + lane] : -1;
  const uint64_t valid = __ballot(id >= 0 && id < p.count);
  // this workgroup's rows
  uint64_t mine = slot == 0 ? __ballot(lane < ROWS && row0 + lane < p.rows) & ~valid : 0;  // rows without an adapter
  const uint64_t plain = mine;
  each_adapter(id, valid, slot, p.slots, [&](int, uint64_t same) __attribute__((always_inline)) { mine |= same; });
  if (!mine) return;

  struct Sixteen {
    T v[16];
  } y[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const T* at = static_cast<const T*>(p.y) + min(row0 + 16 * t + lr, p.rows - 1) * p.ldy;
    if (!(mine >> (16 * t + lr) & 1)) {  // (another slot's)
    } else if (PLAIN || column0 + 64 <= p.n) {
      __builtin_memcpy(&y[t], at + column, sizeof(Sixteen));
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) y[t].v[e] = at[min(column + e, p.n - 1)];
    }
  }
  auto put = [&](int t, uint64_t rows, const f32x4 (&sum)[4]) __attribute__((always_inline)) {
    const int row = 16 * t + lr;
    if (!(rows >> row & 1)) return;
    T* out = static_cast<T*>(p.out) + (row0 + row) * p.n + column;
    // (opaque: else y is waited for and turned into floats before the products)
    u32x4 raw[2];
    __builtin_memcpy(raw, &y[t], sizeof(raw));
    asm volatile("" : "+v"(raw[0]), "+v"(raw[1]));
    Sixteen r;
    __builtin_memcpy(&r, raw, sizeof(r));
#pragma unroll
    for (int e = 0; e < 16; ++e) r.v[e] = (T)((float)r.v[e] + sum[e / 4][e % 4]);
    if (PLAIN || column0 + 64 <= p.n) {
      __builtin_memcpy(out, &r, sizeof(r));
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (column + e < p.n) out[e] = r.v[e];
    }
  };
  const v8* lead = static_cast<const v8*>(p.lead) + row0 / 16 * p.steps * 64 + lane;
  const v8* rest = static_cast<const v8*>(p.rest) + row0 / 16 * p.steps * 64 + lane;
  each_adapter(id, valid, slot, p.slots, [&](int who, uint64_t same) __attribute__((always_inline)) {
    const T* b[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      b[c] = static_cast<const T*>(p.b) + who * p.b_adapter + min(column0 + 16 * (lr >> 2) + 4 * c + (lr & 3), p.n - 1) * p.b_row + 8 * lg;
    v8 w[4], h0[NT], h1[NT];
    int power[NT];  // of the step
    auto load = [&](int s) __attribute__((always_inline)) {
      const int left = p.rank - 32 * s - 8 * lg;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (PLAIN) w[c] = left > 0 ? load_eight<v8>(b[c] + 32 * s) : v8{};
        else w[c] = load_upto<v8>(b[c] + 32 * s, left);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        // (past the last rows there are no operands)
        const int64_t at = (int64_t)min(t, (int)((p.rows - 1 - row0) / 16)) * p.steps * 64 + s * 64;
        h0[t] = lead[at], h1[t] = rest[at];
        if constexpr (__is_same(T, f16_t)) power[t] = p.power[min(row0 + 16 * t + lr, p.rows - 1) * p.steps + s];
      }
    };
    f32x4 sum[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[t][c] = f32x4{0, 0, 0, 0};
    load(0);
#pragma unroll 1
    for (int s = 0; s < p.steps; ++s) {
      v8 w_[4], h0_[NT], h1_[NT];
      int power_[NT];
#pragma unroll
      for (int c = 0; c < 4; ++c) w_[c] = w[c];
#pragma unroll
      for (int t = 0; t < NT; ++t) h0_[t] = h0[t], h1_[t] = h1[t], power_[t] = power[t];
      if (s + 1 < p.steps) load(s + 1);
      f32x4 acc[NT][4];  // (of a step: each has a power of two of its own)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          acc[t][c] = LoraMma<T>::mul(w_[c], h0_[t], f32x4{0, 0, 0, 0});
          acc[t][c] = LoraMma<T>::mul(w_[c], h1_[t], acc[t][c]);
        }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[t][c][e] += __is_same(T, f16_t) ? __builtin_ldexpf(acc[t][c][e], power_[t]) : acc[t][c][e];
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) put(t, same, sum[t]);
  });
  if (plain) {
    const f32x4 zero[4] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
    for (int t = 0; t < NT; ++t) put(t, plain, zero);
  }
}

struct LoraPlan {
  int tiles, parts, slots, hr, lines, steps;  // tiles: of 16 rows of a workgroup
  int64_t parts_bytes, operand_bytes, power_bytes;
};

// Rows of a workgroup, and over how many its adapters are shared out.  Tiles of 64 rows
// read an adapter's weights for fewer of them, but go through each adapter that any of
// the 64 has (fp16, rank 64, rows in order of 4 adapters, 2560 -> 9728: 1024 rows 34 us
// in tiles of 16, 41 of 64; of 7, 9728 -> 2560: 2047 rows 48 and 39; rank 16, 2560 -> 4096,
// 32 adapters in no order: 768 rows 51 and 111, 2047 106 and 185).  Slots for some 128
// workgroups: a tile's adapters in turn are a chain (64 rows of 32 adapters, rank 64,
// 2560 -> 9728: 16 slots 27 us, 4 36, 1 74; 9728 -> 2560: 26, 40 and 113), slots that find
// none cost as well (256 rows of 4: 16 slots 27, 8 21, 4 20; of 32: 28, 25, 30).
//
// Parts of x A^T's sum: of tiles of 64 rows as many as bring 256 workgroups, of at least
// 16 lines each; of 16 rows one up to 96 lines (6144 columns), which needs no join (48
// lines a part: the same).
inline LoraPlan lora_plan(int64_t rows, int64_t k, int64_t rank) {
  LoraPlan q;
  q.tiles = rows > 1024 ? 4 : 1;
  q.slots = q.tiles == 1 ? (int)std::min((int64_t)16, 128 / std::max((int64_t)1, (rows + 15) / 16)) : 1;
  q.hr = (int)(rank + 63) / 64 * 64;
  q.lines = (int)((k + kLine - 1) / kLine);
  q.steps = (int)(rank + 31) / 32;
  int64_t parts;
  if (q.tiles == 1) {
    parts = (q.lines + 95) / 96;
  } else {
    const int64_t groups = (rows + 63) / 64;
    parts = std::min((int64_t)(q.lines + 15) / 16, (256 + groups - 1) / groups);
  }
  q.parts = (int)std::min(parts, (int64_t)16);
  q.parts_bytes = q.parts > 1 ? rows * q.parts * q.hr * 4 : 0;
  q.operand_bytes = (rows + 15) / 16 * q.steps * 1024;
  q.power_bytes = (rows * q.steps * 4 + 15) / 16 * 16;
  return q;
}

template <typename T, int NT, int RT, int W>
void launch_shrink(const LoraArgs& p, hipStream_t s) {
  const dim3 grid((uint32_t)((p.rows + 16 * NT - 1) / (16 * NT)), p.parts, p.slots * ((p.rank + 16 * RT - 1) / (16 * RT)));
  hipLaunchKernelGGL((lora_shrink_kernel<T, NT, RT, W>), grid, dim3(64 * W), 0, s, p);
}

template <typename T, int NT, int W, int NE>
int launch_lora(const LoraArgs& p, hipStream_t s) {
  if (p.count > 0) {
    if (p.rank <= 16) launch_shrink<T, NT, 1, W>(p, s);
    else if (NT == 1 || p.rank <= 32) launch_shrink<T, NT, 2, W>(p, s);
    else if constexpr (NT > 1) launch_shrink<T, NT, 4, W>(p, s);
    if (p.parts > 1)
      hipLaunchKernelGGL((lora_join_kernel<T>), dim3((uint32_t)((p.rows * 4 * p.steps + 255) / 256)), dim3(256), 0, s, p);
  }
  const dim3 grid((uint32_t)((p.rows + 16 * NE - 1) / (16 * NE)), (p.n + 255) / 256, p.slots);
  if (p.rank % 8 == 0 && p.n >= 64) hipLaunchKernelGGL((lora_expand_kernel<T, NE, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((lora_expand_kernel<T, NE, false>), grid, dim3(256), 0, s, p);
  return launch_status();
}

inline bool lora_sizes_ok(int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count) {
  return rows >= 0 && rows <= (1 << 24) && k >= 1 && k <= (1 << 20) && n >= 1 && n <= (1 << 20) && rank >= 1 && rank <= 256 &&
         count >= 0 && count <= (1 << 20) && grid_fits((rows + 31) / 32 * ((n + 255) / 256), 256);
}

}  // namespace tp

using namespace tp;

extern "C" int64_t tp_lora_workspace_bytes(int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count) {
  if (!lora_sizes_ok(rows, k, n, rank, count)) return -1;
  const LoraPlan q = lora_plan(rows, k, rank);
  return count ? q.parts_bytes + 2 * q.operand_bytes + q.power_bytes : 0;
}

extern "C" int tp_lora_add(int dtype, int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t count, const void* x,
                           int64_t ldx, const void* a, int64_t a_adapter, int64_t a_row, const void* b,
                           int64_t b_adapter, int64_t b_row, const int32_t* adapters, const float* scales,
                           const void* y, int64_t ldy, void* out, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  if (dtype != TP_F16 && dtype != TP_BF16) return TP_ERR_BAD_TYPE;
  if (!lora_sizes_ok(rows, k, n, rank, count) || ldx < 0 || ldx > (1 << 24) || a_row < 0 || a_row > (1 << 24) || ldy < 0) return TP_ERR_BAD_DIMS;
  if (rows == 0) return TP_OK;
  if (!x || !y || !out || !adapters || (count && (!a || !b))) return TP_ERR_NULL_POINTER;
  if ((((uintptr_t)x | (uintptr_t)a | (uintptr_t)b | (uintptr_t)y | (uintptr_t)out) & 1) || (((uintptr_t)adapters | (uintptr_t)scales) & 3))
    return TP_ERR_MISALIGNED;
  const int64_t need = tp_lora_workspace_bytes(rows, k, n, rank, count);
  if (need && (!workspace || workspace_bytes < need)) return TP_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return TP_ERR_MISALIGNED;
  const LoraPlan q = lora_plan(rows, k, rank);
  LoraArgs p{};
  p.x = x, p.a = a, p.b = b, p.y = y, p.out = out, p.adapters = adapters, p.scales = scales;
  char* ws = static_cast<char*>(workspace);
  if (need) {
    p.parts_h = reinterpret_cast<float*>(ws), p.lead = ws + q.parts_bytes, p.rest = ws + q.parts_bytes + q.operand_bytes;
    p.power = reinterpret_cast<int*>(ws + q.parts_bytes + 2 * q.operand_bytes);
  }
  p.ldx = ldx, p.ldy = ldy, p.a_adapter = a_adapter, p.a_row = a_row, p.b_adapter = b_adapter, p.b_row = b_row;
  p.rows = rows, p.k = (int)k, p.n = (int)n, p.rank = (int)rank, p.count = (int)count;
  p.parts = q.parts, p.slots = q.slots, p.hr = q.hr, p.lines = q.lines, p.steps = q.steps;
  hipStream_t s = (hipStream_t)stream;
  if (q.tiles == 1) return dtype == TP_F16 ? launch_lora<f16_t, 1, 8, 1>(p, s) : launch_lora<bf16_t, 1, 8, 1>(p, s);
  return dtype == TP_F16 ? launch_lora<f16_t, 4, 8, 2>(p, s) : launch_lora<bf16_t, 4, 8, 2>(p, s);
}
