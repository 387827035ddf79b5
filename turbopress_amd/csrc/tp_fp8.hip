// Product of e4m3 activations and weights with scales per 128 columns:
//
//   y[i, j] = sum_b a_scales[i, b] w_scales[j / 128, b] sum_{c in block b} a[i, c] w[j, c]  (+ bias[j])
//
// A block's inner sum is one matrix instruction (16 x 16 x 128) from zero, and
// one FMA per output multiplies it into fp32 sums; the weights are the
// instructions' rows and the activations their columns, so that a lane's
// outputs share an activation row: one product of scales per lane and block.
// The K order inside a block is the instructions' own for both operands; sums
// over blocks are in a fixed order.
//
// Few rows (fp8_takes_rows): every weight is read once, straight into operand
// registers (bound by HBM: 151936 x 2560, 1 row, 66 us = 5.9 TB/s).  More: tiles
// of both operands are staged in LDS by loads that bypass the registers, bound
// by the matrix cores, LDS and the sums' FMAs together (4096 x 8192 x 8192 256 us
// = 2.15 PFLOP/s; the instructions alone, no staging, sums or LDS reads, ran at
// 3.6) or, of few tiles, by the chain of a tile's blocks (199 x 4096 x 2560 10.3 us:
// 4.9 to begin and end and 0.27 per 128 columns; LDS is busy for 2.9 of them, the
// matrix cores for 1.1).  fp32 outputs of many rows run at a quarter of the matrix
// rate (2048 x 9728 x 2560 116 us against 55 in bf16).
#include "tp_ops_common.h"

#include <algorithm>
#include <type_traits>

namespace tp {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x2 __attribute__((ext_vector_type(2)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

struct Fp8Args {
  const uint8_t *a, *w;
  const float *sa, *sw;
  const void* bias;
  void* y;
  int64_t lda, ldw, ldy, m, n;
  int k, kb;
  int tiles_m, tiles_n;
};

// (cbsz = blgp = 0: both operands e4m3; scale operands 0: the unscaled form)
__device__ __forceinline__ f32x4 mma16(i32x8 w, i32x8 a, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 0, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ void store4(const Fp8Args& g, int64_t i, int64_t j, f32x4 v) {
  if (j >= g.n) return;
  T* y = static_cast<T*>(g.y) + i * g.ldy + j;
  const T* bias = static_cast<const T*>(g.bias) + j;
  if (j + 4 <= g.n) {
    if (g.bias)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += (float)bias[e];
    struct {
      T v[4];
    } r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[e] = (T)v[e];
    __builtin_memcpy(y, &r, sizeof(r));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < g.n) y[e] = (T)(v[e] + (g.bias ? (float)bias[e] : 0.0f));
  }
}

// Operands of a block of 16 rows x 128 columns.  fp16 and bf16 outputs take the
// 8-bit instructions, whose inner sums are good to about 2^-16 of the result
// (measured 1.3e-5 rms, and the same for both of their widths); fp32 outputs
// convert the codes to fp16, exactly, for instructions with fp32 inner sums
// (6e-9), at a quarter of the rate.
template <bool F32>
struct Operand;
template <>
struct Operand<false> {
  i32x8 v;
  __device__ __forceinline__ void set(i32x8 x) { v = x; }
  __device__ __forceinline__ static f32x4 mul(const Operand& w, const Operand& a) {
    return mma16(w.v, a.v, f32x4{0, 0, 0, 0});
  }
};
template <>
struct Operand<true> {
  f16x8 v[4];
  __device__ __forceinline__ void set(i32x8 x) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[2 * q], 1.0f, false);
      const f16x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[2 * q], 1.0f, true);
      const f16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[2 * q + 1], 1.0f, false);
      const f16x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[2 * q + 1], 1.0f, true);
      v[q] = f16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    }
  }
  __device__ __forceinline__ static f32x4 mul(const Operand& w, const Operand& a) {
    f32x4 d{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 4; ++q) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[q], a.v[q], d, 0, 0, 0);
    return d;
  }
};

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------
// A workgroup takes RT tiles of 16 weight rows and all (up to 16 NC)
// activation rows; its waves take every waves-th block of columns, the loads
// of the next one in flight, and their sums are joined through LDS.
// ODD: rows of either operand do not begin on words.
template <typename T, int NC, int RT, bool ODD>
__global__ void __launch_bounds__(NC == 1 ? 1024 : 512) fp8_rows_kernel(const Fp8Args g) {
  using Op = Operand<sizeof(T) == 4>;
  extern __shared__ __attribute__((aligned(16))) char fp8_lds[];
  f32x4* const sums = reinterpret_cast<f32x4*>(fp8_lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * (16 * RT);
  const uint8_t *wp[RT], *ap[NC];
  const float *swp[RT], *sap[NC];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int64_t r = min(row0 + 16 * t + lr, g.n - 1);  // (rows past the end: not stored)
    wp[t] = g.w + r * g.ldw + 32 * lg;
    swp[t] = g.sw + min((row0 + 16 * t) >> 7, (g.n - 1) >> 7) * g.kb;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t i = min((int64_t)(16 * c + lr), g.m - 1);
    ap[c] = g.a + i * g.lda + 32 * lg;
    sap[c] = g.sa + i * g.kb;
  }
  f32x4 acc[RT][NC];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[t][c] = f32x4{0, 0, 0, 0};

  using Codes = std::conditional_t<ODD, Unaligned<8>, i32x8>;
  struct Block {
    Codes w[RT], a[NC];
    float fa[NC], fw[RT];
  };
  auto codes = [&](Codes& x, const uint8_t* p) __attribute__((always_inline)) {
    if constexpr (ODD) x.load(p);
    else __builtin_memcpy(&x, p, 32);
  };
  auto words = [&](const Unaligned<8>& x, const uint8_t* p) __attribute__((always_inline)) {
    const uint32_t s = (uint32_t)(uintptr_t)p & 3;
    i32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = (int)x.word(e, s);
    return r;
  };
  auto aligned = [&](const Codes& x, const uint8_t* p) __attribute__((always_inline)) {
    if constexpr (ODD) return words(x, p);
    else return x;
  };
  auto load = [&](Block& x, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < RT; ++t) codes(x.w[t], wp[t] + 128 * b);
#pragma unroll
    for (int c = 0; c < NC; ++c) codes(x.a[c], ap[c] + 128 * b), x.fa[c] = sap[c][b];
#pragma unroll
    for (int t = 0; t < RT; ++t) x.fw[t] = swp[t][b];
  };
  auto add = [&](const Block& x) __attribute__((always_inline)) {
    Op a[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) a[c].set(aligned(x.a[c], ap[c]));
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      Op w;
      w.set(aligned(x.w[t], wp[t]));
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[t][c] += Op::mul(w, a[c]) * (x.fa[c] * x.fw[t]);
    }
  };
  const int whole = g.k >> 7;  // blocks without a tail
  if (wave < whole) {
    Block x, y;
    load(x, wave);
    for (int b = wave; b < whole; b += waves) {
      // (past the last: the first again, not used)
      load(y, b + waves < whole ? b + waves : wave);
      add(x);
      x = y;
    }
  }
  if (whole < g.kb && wave == whole % waves) {
    const int left = g.k - 128 * whole - 32 * lg;  // columns of this lane's 32
    Block x;
    auto rest = [&](Codes& x, const uint8_t* p) __attribute__((always_inline)) {
      Unaligned<8> u;
      u.load_first(p, min(left, 32));
      if constexpr (ODD) x = u;
      else x = words(u, p);
    };
#pragma unroll
    for (int t = 0; t < RT; ++t) rest(x.w[t], wp[t] + 128 * whole), x.fw[t] = swp[t][whole];
#pragma unroll
    for (int c = 0; c < NC; ++c) rest(x.a[c], ap[c] + 128 * whole), x.fa[c] = sap[c][whole];
    add(x);
  }

#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int c = 0; c < NC; ++c) sums[(wave * RT * NC + t * NC + c) * 64 + lane] = acc[t][c];
  __syncthreads();
  for (int p = wave; p < RT * NC; p += waves) {
    f32x4 y = sums[p * 64 + lane];
    for (int x = 1; x < waves; ++x) y += sums[(x * RT * NC + p) * 64 + lane];
    const int t = p / NC, c = p - t * NC;
    const int64_t i = 16 * c + lr;
    if (i < g.m) store4<T>(g, i, row0 + 16 * t + 4 * lg, y);
  }
}

// ---------------------------------------------------------------------------
// more rows
// ---------------------------------------------------------------------------
// A workgroup of WK teams of WN x WM waves, a wave TN x TM blocks of 16 weight
// rows x 16 activation rows; the teams share the columns' blocks, each in LDS of
// its own, and their sums are joined at the end.  A team's LDS holds kBufs stages of 128 columns; a row's eight 16-byte
// chunks are stored in the order c ^ (row & 7), so that the rows that a lane
// group reads at one chunk fall on distinct banks (a load to LDS writes lane
// after lane, so the lanes' global addresses are permuted).
template <int WN, int WM, int TN, int TM, int WK>
struct TileShape {
  static constexpr int kWaves = WN * WM;  // of a team
  static constexpr int kBN = 16 * WN * TN, kBM = 16 * WM * TM;
  static constexpr int kStage = (kBN + kBM) * 128;
  static constexpr int kBufs = WK <= 2 && 4 * kStage <= 64 * 1024 ? 4 : WK == 1 && 3 * kStage <= 72 * 1024 ? 3 : 2;
  // scales of kSB stages, [row][kSB] activations' and [64 / kSB][kSB] weights': of
  // those in use, those arriving, and those that stages ahead of the block call for
  static constexpr int kScales = kBufs * kStage;
  static constexpr int kSB = WK * (kScales + 3 * (kBM * 32 + 256)) <= 160 * 1024 ? 8 : 4;
  static constexpr int kScaleBuf = kBM * 4 * kSB + 256;
  static constexpr int kTeam = kScales + 3 * kScaleBuf, kLds = WK * kTeam;  // bytes of a team, of the workgroup
  static constexpr int kWLoads = kBN / 8 / kWaves, kALoads = kBM / 8 / kWaves;  // 1 KB pieces (8 rows) of a wave
  static constexpr int kLoads = kWLoads + kALoads + 2;
  static_assert(kBN % (8 * kWaves) == 0 && kBM % (8 * kWaves) == 0 && kBM % 64 == 0 && 64 * kWaves >= kBM && kLds <= 160 * 1024, "");
};

template <int N>
__device__ __forceinline__ void wait_vm() {
  __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (uint32_t)std::min<int64_t>(bytes, 0xfffffff0), 0x00020000);
}

constexpr int kLate = 3;  // products between one and its sums

template <typename T, int WN, int WM, int TN, int TM, int WK>
__global__ void __launch_bounds__(64 * WN * WM * WK, WK > 2 ? 1 : 2) fp8_tile_kernel(const Fp8Args g) {
  using S = TileShape<WN, WM, TN, TM, WK>;
  using Op = Operand<sizeof(T) == 4>;
  constexpr int BN = S::kBN, BM = S::kBM, NBUF = S::kBufs;
  extern __shared__ __attribute__((aligned(16))) char fp8_lds[];
  const int lane = threadIdx.x & 63, wave0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = WK == 1 ? 0 : wave0 / S::kWaves, wave = WK == 1 ? wave0 : wave0 % S::kWaves;
  const int wn = wave % WN, wm = wave / WN;
  char* const lds = fp8_lds + team * S::kTeam;
  // the team's blocks: b0 .. b0 + blocks - 1, the last team's up to the last one
  // (blocks below 0, of the first teams, are zeros)
  const int blocks = (g.kb + WK - 1) / WK, b0 = g.kb - (WK - team) * blocks;

  // each XCD (blockIdx % 8) takes a contiguous run of tiles, activation tiles
  // fastest: they share a weight tile in its L2
  const int total = (int)gridDim.x, q8 = total >> 3, r8 = total & 7, xcd = (int)blockIdx.x & 7;
  const int tile = xcd * q8 + min(xcd, r8) + ((int)blockIdx.x >> 3);
  const int tn = tile / g.tiles_m, tm = tile - tn * g.tiles_m;
  const int64_t n0 = (int64_t)tn * BN, m0 = (int64_t)tm * BM;

  // Reads past the last row's columns, rounded up to 16, return zero (its
  // 16-byte chunks hold a byte of the row each, so none is outside memory).
  // The scalar offset is the column's alone, below the record count: the range
  // check subtracts it.
  const int64_t kr = (g.k + 15) & ~15;
  const __amdgpu_buffer_rsrc_t wrs = rows_rsrc(g.w + n0 * g.ldw, (std::min<int64_t>(BN, g.n - n0) - 1) * g.ldw + kr);
  const __amdgpu_buffer_rsrc_t ars = rows_rsrc(g.a + m0 * g.lda, (std::min<int64_t>(BM, g.m - m0) - 1) * g.lda + kr);
  const __amdgpu_buffer_rsrc_t sars = rows_rsrc(g.sa + m0 * g.kb, std::min<int64_t>(BM, g.m - m0) * g.kb * 4);
  const int64_t nb0 = n0 >> 7;  // weight blocks of the tile
  const __amdgpu_buffer_rsrc_t swrs = rows_rsrc(g.sw + nb0 * g.kb, (((g.n - 1) >> 7) - nb0 + 1) * g.kb * 4);
  const uint32_t lrow = lane >> 3, chunk = ((lane & 7) ^ lrow) * 16;  // of an 8-row piece
  const uint32_t wv = (uint32_t)(8 * wave * S::kWLoads + lrow) * (uint32_t)g.ldw + chunk;
  const uint32_t av = (uint32_t)(8 * wave * S::kALoads + lrow) * (uint32_t)g.lda + chunk;
  // Scales go to LDS too (a scalar load would make every LDS wait a full one),
  // those of SB = 8 (4) blocks together: a load takes 8 rows x 8 blocks, 32 bytes
  // of a row (64 rows x 1 block at a time, 64 pieces of memory in one load, took
  // as long as all operands).  With stage SB q + j goes the j-th SB-th part of
  // the scales of blocks SB (q + 1) .. SB (q + 1) + SB - 1.
  constexpr int SB = S::kSB, kRows = 64 / SB;  // rows of a load
  const uint32_t srow = kRows * (wave % (BM / 64)) + lane / SB;
  const uint32_t sav = srow * (uint32_t)g.kb * 4u, swv = (lane / SB) * (uint32_t)g.kb * 4u;
  // (j and i count the team's blocks)
  auto stage_scales = [&](int j, int i, int ring) __attribute__((always_inline)) {  // its blocks i .. i + SB - 1
    char* p = lds + S::kScales + ring * S::kScaleBuf;
    const int b = b0 + i + (int)(lane % SB);
    // (blocks before the first and past the last: zeros)
    const uint32_t at = (uint32_t)b >= (uint32_t)g.kb ? 0x80000000u : 4u * b;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        sars, (__attribute__((address_space(3))) void*)(p + (j * (BM / SB) + kRows * (wave % (BM / 64))) * 4 * SB), 4,
        at + sav + (uint32_t)(j * (BM / SB)) * (uint32_t)g.kb * 4u, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(swrs, (__attribute__((address_space(3))) void*)(p + BM * 4 * SB), 4, at + swv, 0, 0,
                                             0);
  };
  int ring = 1;  // where the next scales go
  auto stage = [&](int i, int buf) __attribute__((always_inline)) {
    char* p = lds + buf * S::kStage;
    const int b = b0 + i, bc = min(max(b, 0), g.kb - 1);
    // chunks past the columns, and stages that are not, load nothing: zeros
    const uint32_t past = b < 0 || 128 * b + (int)chunk >= kr ? 0x80000000u : 0u;
    stage_scales(i & (SB - 1), (i & -SB) + SB, ring);
    ring = (i & (SB - 1)) == SB - 1 ? (ring == 2 ? 0 : ring + 1) : ring;
#pragma unroll
    for (int x = 0; x < S::kWLoads; ++x)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wrs, (__attribute__((address_space(3))) void*)(p + (wave * S::kWLoads + x) * 1024), 16,
          (wv | past) + (uint32_t)(8 * x) * (uint32_t)g.ldw, 128u * bc, 0, 0);
#pragma unroll
    for (int x = 0; x < S::kALoads; ++x)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          ars, (__attribute__((address_space(3))) void*)(p + BN * 128 + (wave * S::kALoads + x) * 1024), 16,
          (av | past) + (uint32_t)(8 * x) * (uint32_t)g.lda, 128u * bc, 0, 0);
  };
  // The bytes past the columns of the last stage's last chunk, which hold
  // anything, are zeroed (by the wave that loaded them).
  auto zero_rest = [&](int buf) __attribute__((always_inline)) {
    const int in = g.k - (128 * (g.kb - 1) + (int)chunk);  // columns of this lane's chunk
    if (team == WK - 1 && in > 0 && in < 16) {
      u32x4 keep;
#pragma unroll
      for (int e = 0; e < 4; ++e) keep[e] = in >= 4 * e + 4 ? ~0u : in <= 4 * e ? 0u : (1u << (8 * (in - 4 * e))) - 1;
      u32x4* p = reinterpret_cast<u32x4*>(lds + buf * S::kStage) + lane;
#pragma nounroll
      for (int x = 0; x < S::kWLoads + S::kALoads; ++x)
        p[64 * (x < S::kWLoads ? wave * S::kWLoads + x : BN / 8 + wave * S::kALoads + x - S::kWLoads)] &= keep;
    }
  };

  // operand: columns 32 lg .. + 31 of row lr of 16
  const int lr = lane & 15, lg = lane >> 4;
  const uint32_t o0 = lr * 128 + (((2 * lg) ^ (lr & 7)) << 4), o1 = lr * 128 + (((2 * lg + 1) ^ (lr & 7)) << 4);
  auto operand = [&](const char* rows) __attribute__((always_inline)) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(rows + o0), hi = *reinterpret_cast<const u32x4*>(rows + o1);
    Op op;
    op.set(i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]});
    return op;
  };
  f32x4 acc[TN][TM], d[kLate + 1];
  // Scales: of the products in d; of the current block, apart.  A wave's weight
  // rows lie in one block of 128 where 16 TN divides 128, else in up to 3, whose
  // first ends at the wave's row `edge`.
  constexpr bool kOneBlock = 128 % (16 * TN) == 0;
  constexpr int kWS = kOneBlock ? 1 : 3;
  const int wrow = (int)(n0 & 127) + wn * 16 * TN, wblk = kOneBlock ? (wn * 16 * TN) >> 7 : wrow >> 7;
  const int edge = 128 - (wrow & 127);
  float f[TM], fa[TM], fw[kWS];
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int c = 0; c < TM; ++c) acc[t][c] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int x = 0; x <= kLate; ++x) d[x] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int c = 0; c < TM; ++c) f[c] = 0.0f;
  constexpr int kAhead = TN * TM >= 40 ? 2 : TN < 4 ? TN : 4;  // weight operands in registers, read kAhead - 1 groups ahead
  Op a[TM], w[kAhead];
  // what a block's first products need
  auto first = [&](int i, int buf, int ring) __attribute__((always_inline)) {
    const char* p = lds + buf * S::kStage;
    const float* sl = reinterpret_cast<const float*>(lds + S::kScales + ring * S::kScaleBuf) + (i & (SB - 1));
    // (the order of their use; the scales' product is formed where it is used)
    w[0] = operand(p + wn * 16 * TN * 128);
#pragma unroll
    for (int c = 0; c < TM; ++c) a[c] = operand(p + BN * 128 + (wm * TM + c) * 16 * 128);
#pragma unroll
    for (int t = 1; t < kAhead - 1; ++t) w[t] = operand(p + (wn * TN + t) * 16 * 128);
#pragma unroll
    for (int x = 0; x < kWS; ++x) fw[x] = sl[(BM + wblk + x) * SB];
#pragma unroll
    for (int c = 0; c < TM; ++c) fa[c] = sl[(wm * 16 * TM + 16 * c + lr) * SB];
  };
  // Product n of a block is block (n / TM, n % TM); its sums follow kLate products
  // later, the last ones' in the next block.
  auto sums = [&](int n) __attribute__((always_inline)) {
    const int t = n / TM, c = n % TM;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][c][e] = fmaf(d[n % (kLate + 1)][e], f[c], acc[t][c][e]);
  };
  static_assert(TN * TM % (kLate + 1) == 0 && (kOneBlock || TM == kLate + 1), "products keep their place in d, scales of a group are formed in its block");

  // A block of 128 columns.  sched_barrier keeps the order of products, sums and
  // reads: left alone the scheduler gathers the reads, and waits for each
  // group's products.
  auto block = [&](int buf) __attribute__((always_inline)) {
    const char* wl = lds + buf * S::kStage + wn * 16 * TN * 128;
#pragma unroll
    for (int n = 0; n < TN * TM; ++n) {
      const int t = n / TM, c = n % TM;
      if (c == 0 && t + kAhead - 1 < TN) w[(t + kAhead - 1) % kAhead] = operand(wl + (t + kAhead - 1) * 16 * 128);
      d[n % (kLate + 1)] = Op::mul(w[t % kAhead], a[c]);
      // the scales of product n - kLate: its row of blocks' first one is next
      const int m = (n + TN * TM - kLate) % (TN * TM);
      if (m % TM == 0 && (m == 0 || !kOneBlock)) {
        const int r = 16 * (m / TM);
        const float ws = kOneBlock ? fw[0] : r < edge ? fw[0] : r < edge + 128 ? fw[kWS / 2] : fw[kWS - 1];
#pragma unroll
        for (int x = 0; x < TM; ++x) f[x] = fa[x] * ws;
      }
      sums(m);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto meet = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
  };

#pragma unroll
  for (int j = 0; j < SB; ++j) stage_scales(j, 0, 0);
#pragma unroll
  for (int s = 0; s < NBUF; ++s) stage(s, s);
  wait_vm<(NBUF - 1) * S::kLoads>();
  meet();
  first(0, 0, 0);
  int buf = 0, used = 0;  // used: where the block's scales are
  for (int i = 0; i + 1 < blocks; ++i) {
    block(buf);
    // With the last products under way the next stage is complete (its loads
    // were issued a block ago) and every wave has read this one: its buffer
    // takes the next loads, and the next block's first operands are read.
    wait_vm<(NBUF - 2) * S::kLoads>();
    meet();
    stage(i + NBUF, buf);
    buf = buf + 1 == NBUF ? 0 : buf + 1;
    used = (i & (SB - 1)) == SB - 1 ? (used == 2 ? 0 : used + 1) : used;
    first(i + 1, buf, used);
  }
  if (g.k & 15) {
    zero_rest(buf);
    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    meet();
    first(blocks - 1, buf, used);
  }
  block(buf);
  wait_vm<0>();  // (no load to LDS may be in flight when the workgroup ends)
#pragma unroll
  for (int n = TN * TM - kLate; n < TN * TM; ++n) sums(n);
  // (the sums end here: sunk into the stores' branches they spill)
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int c = 0; c < TM; ++c) __asm__ volatile("" : "+v"(acc[t][c]));

  // Out through LDS, 16 activation rows of a wave at a time (a lane holds row lr
  // and weight rows 4 lg .. + 3 of a block): whole rows of the wave's 16 TN
  // columns in 16-byte stores.  Stored as they lie, 8 bytes a lane over 16 rows,
  // a tile of 256 x 256 took about 15 us more.
  meet();
  if constexpr (WK > 1) {
    // the teams' sums, in their order
    f32x4* const sums_lds = reinterpret_cast<f32x4*>(fp8_lds) + lane;
    static_assert((WK - 1) * S::kWaves * TN * TM * 1024 <= S::kLds, "");
    if (team > 0)
#pragma unroll
      for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int c = 0; c < TM; ++c) sums_lds[((((team - 1) * S::kWaves + wave) * TN + t) * TM + c) * 64] = acc[t][c];
    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    meet();
    if (team > 0) return;
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int c = 0; c < TM; ++c) {
#pragma unroll
        for (int x = 0; x < WK - 1; ++x) acc[t][c] += sums_lds[(((x * S::kWaves + wave) * TN + t) * TM + c) * 64];
      }
  }
  constexpr int kPer = 16 / sizeof(T);                   // elements of a store
  constexpr int kPitch = 16 * TN * (int)sizeof(T) + 16;  // of a row in LDS
  constexpr int kChunks = 16 * TN / kPer;                // stores of a row
  struct Out {
    T v[kPer];
  };
  constexpr int kOut = WK == 1 ? 0 : (WK - 1) * S::kWaves * TN * TM * 1024;  // (behind the sums: other waves still read them)
  char* const ol = fp8_lds + kOut + wave * 16 * kPitch;
  static_assert(kOut + S::kWaves * 16 * kPitch <= S::kLds, "");
  const int64_t j0 = n0 + wn * 16 * TN;
  const T* bias = static_cast<const T*>(g.bias);
#pragma unroll
  for (int c = 0; c < TM; ++c) {
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      struct {
        T v[4];
      } o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t j = j0 + 16 * t + 4 * lg + e;
        o.v[e] = (T)(acc[t][c][e] + (bias && j < g.n ? (float)bias[j] : 0.0f));
      }
      __builtin_memcpy(ol + lr * kPitch + (16 * t + 4 * lg) * (int)sizeof(T), &o, sizeof(o));
    }
    wave_lds_fence();
    const int64_t i0 = m0 + wm * 16 * TM + 16 * c;
    T* y = static_cast<T*>(g.y) + i0 * g.ldy + j0;
#pragma unroll
    for (int x = 0; x < 16 * kChunks / 64; ++x) {
      const int id = 64 * x + lane, row = id / kChunks, j = (id - row * kChunks) * kPer;
      const u32x4 w = *reinterpret_cast<const u32x4*>(ol + row * kPitch + j * (int)sizeof(T));
      if (i0 + row < g.m) {
        if (j0 + j + kPer <= g.n) {
          __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any*>(y + (int64_t)row * g.ldy + j));
        } else {
          const Out o = __builtin_bit_cast(Out, w);
#pragma unroll
          for (int e = 0; e < kPer; ++e)
            if (j0 + j + e < g.n) y[(int64_t)row * g.ldy + j + e] = o.v[e];
        }
      }
    }
    wave_lds_fence();
  }
}

// Rows of any alignment, of one operand or of both, copied to rows of `ld` bytes
// (a multiple of 16): 16 lanes copy 1 KB of a row, 4 chunks each.
struct Fp8Copies {
  const uint8_t* src[2];
  uint8_t* dst[2];
  int64_t from[2], rows[2];  // row strides of the sources, rows (none: aligned)
  int64_t ld;
  int k;
};

__global__ void __launch_bounds__(256) fp8_align_kernel(Fp8Copies g) {
  int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool second = r >= g.rows[0];
  if (second) r -= g.rows[0];
  if (second && r >= g.rows[1]) return;
  const uint8_t* const src = g.src[second] + r * g.from[second];
  uint8_t* const dst = g.dst[second] + r * g.ld;
  const int first = (int)blockIdx.y * 1024 + (int)(threadIdx.x & 15) * 16;
  Unaligned<4> v[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int c = first + 256 * x;
    if (c + 16 <= g.k) v[x].load(src + c);
    else v[x].load_first(src + c, g.k - c);
  }
  const uint32_t s = (uint32_t)(uintptr_t)src & 3;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (first + 256 * x < g.k)
      *reinterpret_cast<u32x4*>(dst + first + 256 * x) = u32x4{v[x].word(0, s), v[x].word(1, s), v[x].word(2, s), v[x].word(3, s)};
}

constexpr int64_t kMaxLd = (int64_t)1 << 36;  // (times 2^26 rows: offsets of 64 bits)

bool fp8_sizes_ok(int64_t m, int64_t n, int64_t k) {
  return m >= 0 && n >= 0 && k >= 1 && m <= (1 << 24) && n <= (1 << 26) && k <= (1 << 20);
}

// Rows that the tiles load as they lie: 16-byte pieces, 32-bit offsets inside a
// tile (320 rows of up to 2^22 bytes).  Others are copied for them; the rows
// kernel, whose offsets have 64 bits, takes any.
bool fp8_rows_tiled(const void* p, int64_t ld) { return ((ld | (int64_t)(uintptr_t)p) & 15) == 0 && ld <= (1 << 22); }

template <typename T, int NC, int RT, bool ODD>
void launch_rows(const Fp8Args& g, int waves, hipStream_t s) {
  const int64_t groups = (g.n + 16 * RT - 1) / (16 * RT);
  const int lds = waves * RT * NC * 64 * 16;
  if (lds > 64 * 1024) allow_dynamic_lds(reinterpret_cast<const void*>(&fp8_rows_kernel<T, NC, RT, ODD>), 0);
  hipLaunchKernelGGL((fp8_rows_kernel<T, NC, RT, ODD>), dim3((uint32_t)groups), dim3(64 * waves), lds, s, g);
}

// Whether a call takes the rows kernel.  us at (n, k), rows kernel against the
// fastest tiles:
//   32 rows  1024, 1024: 4.5 / 6.0   4096, 2560: 7.2 / 9.5   2560, 9728: 17.9 / 23.3   9728, 2560: 15.2 / 10.0
//   64 rows  4096, 2560: 10.3 / 10.1  2560, 9728: 28.8 / 24.0   9728, 2560: 20.2 / 10.0
// so 17..32 rows take it for up to 6144 weight rows (the tiles' time is their
// chain of blocks until their count fills the GPU), more rows never.  Operands
// that are not fp8_rows_tiled are copied for the tiles: 32 rows, 7000, 100: 3.8
// / 9.4  16384, 1000: 11.4 / 19.2  16000, 5003: 57.6 / 51.4, so they take it up to
// 32 MB of weights, halfway.
bool fp8_takes_rows(int64_t m, int64_t n, int64_t k, bool tiled) {
  return m <= 16 || (m <= 32 && (n <= 6144 || (!tiled && n * k <= (32 << 20))));
}

// How the rows kernel cuts a call.
struct RowsPlan {
  int waves, tiles;  // that share a tile's columns; tiles of a workgroup
};

// 8 waves share a tile's columns (4 / 8 / 16 waves, 1 row: 4096 x 2560 5.5 / 4.6 /
// 4.9 us, 2560 x 9728 12.6 / 8.4 / 8.3); two tiles per workgroup where that leaves
// two workgroups per CU (1 / 2 tiles, 1 row: 151936 x 2560 76.9 / 66.8 us, 16384 x
// 1000 8.5 / 7.4, 9728 x 2560 7.8 / 8.5)
inline RowsPlan rows_plan(int64_t m, int64_t n, int64_t kb, int64_t cus) {
  RowsPlan p{8, m <= 16 && (n + 15) / 16 >= 4 * cus ? 2 : 1};
  while (p.waves > 1 && p.waves > kb) p.waves /= 2;
  return p;
}

template <typename T>
int launch_rows_for(const Fp8Args& g, hipStream_t s) {
  const RowsPlan p = rows_plan(g.m, g.n, g.kb, device_cu_count());
  const int waves = p.waves;
  const bool two = p.tiles == 2;
  const bool odd = (((uintptr_t)g.a | (uintptr_t)g.w | g.lda | g.ldw) & 3) != 0;
  if (g.m <= 16) {
    if (two && odd) launch_rows<T, 1, 2, true>(g, waves, s);
    else if (two) launch_rows<T, 1, 2, false>(g, waves, s);
    else if (odd) launch_rows<T, 1, 1, true>(g, waves, s);
    else launch_rows<T, 1, 1, false>(g, waves, s);
  } else if (odd) {
    launch_rows<T, 2, 1, true>(g, waves, s);
  } else {
    launch_rows<T, 2, 1, false>(g, waves, s);
  }
  return launch_status();
}

template <typename T, int WN, int WM, int TN, int TM, int WK = 1>
int launch_tiles(Fp8Args g, hipStream_t s) {
  using S = TileShape<WN, WM, TN, TM, WK>;
  g.tiles_m = (int)((g.m + S::kBM - 1) / S::kBM), g.tiles_n = (int)((g.n + S::kBN - 1) / S::kBN);
  const int64_t total = (int64_t)g.tiles_m * g.tiles_n;
  if (!grid_fits(total, 64 * S::kWaves * WK)) return TP_ERR_BAD_DIMS;
  if (S::kLds > 64 * 1024) allow_dynamic_lds(reinterpret_cast<const void*>(&fp8_tile_kernel<T, WN, WM, TN, TM, WK>), 0);
  hipLaunchKernelGGL((fp8_tile_kernel<T, WN, WM, TN, TM, WK>), dim3((uint32_t)total), dim3(64 * S::kWaves * WK), S::kLds, s, g);
  return launch_status();
}

// Rounds of workgroups over the GPU times what a round takes, us: per block of
// 128 columns, with one workgroup on a CU and with as many as it holds, and 4 to
// begin and end.  Times of the shapes in their order (picks in brackets):
//   2048 x 9728 x 2560 (rows, weight rows, columns)  [63] 82 74 78 98 128 171
//   4096 x 8192 x 8192  289 [262] 298 335 427 648 723
//   1024 x 2560 x 9728  150 126 106 69 [59] 70 78
//   512 x 4096 x 2560   50 39 33 21 14.8 [14.3] 18.5
//   256 x 2560 x 9728   146 122 100 61 40 29 [24.0]
//   199 x 4096 x 2560   49 39 33 20 14.3 10.8 [10.3]
struct Fp8Shape {
  int n, m, teams, per_cu;
  double one, full;
};
constexpr Fp8Shape kFp8Shapes[] = {{320, 256, 1, 1, 2.4, 2.4}, {256, 256, 1, 1, 1.9, 1.9},   {256, 192, 1, 1, 1.6, 1.6},
                                   {128, 128, 1, 2, 0.78, 1.15}, {128, 64, 1, 2, 0.5, 0.77}, {64, 64, 1, 2, 0.35, 0.5},
                                   {64, 64, 2, 1, 0.28, 0.28}};

inline int pick_tiles(bool f32, int64_t m, int64_t n, int64_t kb, int64_t cus) {
  // (fp32 outputs: the operands of the largest, converted, do not fit the registers)
  int best = f32 ? 3 : 0;
  double least = 0;
  for (int x = best, first = best; x < 7; ++x) {
    const Fp8Shape& p = kFp8Shapes[x];
    const int64_t t = ((m + p.m - 1) / p.m) * ((n + p.n - 1) / p.n);
    const double c = t <= cus ? kb * p.one + 4 : (double)((t + cus * p.per_cu - 1) / (cus * p.per_cu)) * (kb * p.full + 4);
    if (x == first || c < least) best = x, least = c;
  }
  return best;
}

template <typename T>
int launch_tiles_for(const Fp8Args& g, hipStream_t s) {
  const int best = pick_tiles(sizeof(T) == 4, g.m, g.n, g.kb, device_cu_count());
  if constexpr (sizeof(T) != 4) {
    if (best == 0) return launch_tiles<T, 2, 4, 10, 4>(g, s);
    if (best == 1) return launch_tiles<T, 2, 4, 8, 4>(g, s);
    if (best == 2) return launch_tiles<T, 2, 4, 8, 3>(g, s);
  }
  if (best == 3) return launch_tiles<T, 2, 2, 4, 4>(g, s);
  if (best == 4) return launch_tiles<T, 2, 2, 4, 2>(g, s);
  if (best == 5) return launch_tiles<T, 2, 2, 2, 2>(g, s);
  return launch_tiles<T, 2, 2, 2, 2, 2>(g, s);
}

template <typename T>
int launch_fp8(const Fp8Args& g, bool rows, hipStream_t s) {
  return rows ? launch_rows_for<T>(g, s) : launch_tiles_for<T>(g, s);
}

int64_t align_bytes(int64_t rows, int64_t k) { return rows * ((k + 15) & ~(int64_t)15); }

}  // namespace tp

using namespace tp;

extern "C" int64_t tp_fp8_workspace_bytes(int64_t m, int64_t n, int64_t k, const uint8_t* a, int64_t lda,
                                          const uint8_t* w, int64_t ldw) {
  if (!fp8_sizes_ok(m, n, k)) return -1;
  const bool tiled = fp8_rows_tiled(a, lda) && fp8_rows_tiled(w, ldw);
  if (m == 0 || n == 0 || fp8_takes_rows(m, n, k, tiled)) return 0;
  return (fp8_rows_tiled(a, lda) ? 0 : align_bytes(m, k)) + (fp8_rows_tiled(w, ldw) ? 0 : align_bytes(n, k));
}

extern "C" int tp_fp8_plan(int dtype, int64_t m, int64_t n, int64_t k, int tiled, int cus, int64_t* out) {
  if (!out) return TP_ERR_NULL_POINTER;
  for (int i = 0; i < 5; ++i) out[i] = 0;
  if (!dtype_ok(dtype)) return TP_ERR_BAD_TYPE;
  if (!fp8_sizes_ok(m, n, k) || m == 0 || n == 0 || cus < 1) return TP_ERR_BAD_DIMS;
  const int64_t kb = (k + 127) / 128;
  if (fp8_takes_rows(m, n, k, tiled != 0)) {
    const RowsPlan p = rows_plan(m, n, kb, cus);
    out[0] = 1, out[1] = 16 * p.tiles, out[2] = m <= 16 ? 16 : 32, out[3] = p.waves;
  } else {
    const Fp8Shape& p = kFp8Shapes[pick_tiles(dtype == TP_F32, m, n, kb, cus)];
    out[1] = p.n, out[2] = p.m, out[3] = p.teams;
  }
  out[4] = ((n + out[1] - 1) / out[1]) * ((m + out[2] - 1) / out[2]);
  return TP_OK;
}

extern "C" int tp_fp8_linear(int dtype, int64_t m, int64_t n, int64_t k, const uint8_t* a, int64_t lda,
                             const float* a_scales, const uint8_t* w, int64_t ldw, const float* w_scales,
                             const void* bias, void* y, int64_t ldy, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  if (!dtype_ok(dtype)) return TP_ERR_BAD_TYPE;
  if (!fp8_sizes_ok(m, n, k) || lda < k || ldw < k || ldy < n || lda > kMaxLd || ldw > kMaxLd) return TP_ERR_BAD_DIMS;
  if (m == 0 || n == 0) return TP_OK;
  if (!a || !a_scales || !w || !w_scales || !y) return TP_ERR_NULL_POINTER;
  const uintptr_t mask = dtype_bytes(dtype) - 1;
  if ((((uintptr_t)a_scales | (uintptr_t)w_scales) & 3) || (((uintptr_t)bias | (uintptr_t)y) & mask)) return TP_ERR_MISALIGNED;
  const bool rows = fp8_takes_rows(m, n, k, fp8_rows_tiled(a, lda) && fp8_rows_tiled(w, ldw));
  const int64_t need = tp_fp8_workspace_bytes(m, n, k, a, lda, w, ldw);
  if (need > 0 && (!workspace || workspace_bytes < need)) return TP_ERR_WORKSPACE;
  if (need > 0 && ((uintptr_t)workspace & 15)) return TP_ERR_MISALIGNED;
  hipStream_t s = (hipStream_t)stream;
  if (need > 0) {
    Fp8Copies c{{a, w}, {nullptr, nullptr}, {lda, ldw}, {0, 0}, (k + 15) & ~(int64_t)15, (int)k};
    uint8_t* free = static_cast<uint8_t*>(workspace);
    auto align = [&](int x, const uint8_t*& p, int64_t& from, int64_t rows) {
      if (fp8_rows_tiled(p, from)) return;
      c.dst[x] = free, c.rows[x] = rows;
      p = free, from = c.ld;
      free += rows * c.ld;
    };
    align(0, a, lda, m);
    align(1, w, ldw, n);
    const dim3 grid((uint32_t)((c.rows[0] + c.rows[1] + 15) / 16), (uint32_t)((k + 1023) / 1024));
    hipLaunchKernelGGL(fp8_align_kernel, grid, dim3(256), 0, s, c);
  }
  Fp8Args g{a, w, a_scales, w_scales, bias, y, lda, ldw, ldy, m, n, (int)k, (int)((k + 127) / 128), 0, 0};
  if (dtype == TP_F16) return launch_fp8<f16_t>(g, rows, s);
  if (dtype == TP_BF16) return launch_fp8<bf16_t>(g, rows, s);
  return launch_fp8<float>(g, rows, s);
}
