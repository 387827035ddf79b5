// Attention of one new token per sequence over a paged cache, or of a tree of up
// to 64 that are drafted (TREE).  With the running
// maximum m and sum l of a softmax, a block of tokens takes a state (m, l, o) to
//
//   m' = max(m, max_t s_t),  l' = l e^(m - m') + sum_t e^(s_t - m'),
//   o' = o e^(m - m') + sum_t e^(s_t - m') v_t
//
// and two states join in the same way, so a sequence may be cut anywhere.
// Keys and values are read once, 4 * (query heads per cache head) flops for
// each of their elements: bound by HBM (8 heads of 128: 64 sequences x 8192
// tokens 352 us = 6.1 TB/s, 1 x 131072 99 us = 5.4 with its start and join; 1 x
// 577 9.2 us, the chain of lengths, pages, keys and join).
//
// Work: 128 tokens (256 of up to 64 columns) of one (sequence, cache head) are a
// unit, for up to 16 query heads: more of them read keys and values again (16 x
// 8192 tokens of one cache head of 128: 16 query heads 25 us, 32 32, 48 47).  A grid of as many
// workgroups as the GPU holds takes equal runs of the list of all units, so
// uneven sequences, one long one and many short ones all fill it; the lengths
// are only known on the device, and every workgroup finds its run by a scan of
// them.  A workgroup that ends inside a (sequence, head) leaves its state in
// the workspace; the last one of that head to finish joins them.
//
// A wave takes 32 tokens at a time: S^T = K Q^T with the keys as the matrix
// instructions' rows, straight from memory into the operand registers, so that
// a lane holds one query head and its softmax needs no LDS; O^T = V^T P^T takes
// the probabilities from the registers where S^T left them, and V through a
// wave's own piece of LDS, read transposed.  Loads of the next 32 tokens are in
// flight meanwhile.
//
// TREE: new token j of a sequence is token length + j of its cache, and sees those
// before the length and, of the new ones, the bits of its mask.  A row is a (new
// token, query head) of the cache head, up to 64 rows share what a workgroup reads,
// and which of them see a token is asked only in the tiles where they differ.  4
// flops for each element and row: from 64 rows on the exponentials, products and the
// waits between them bound it, not HBM (16 new tokens, 32 query heads on 8 of 128
// columns: 131072 tokens 131 + 8 us of the join = 3.9 TB/s; 13 of 32 sequences of 0 to
// 8191 143 + 10; 64 new tokens of 16 sequences of 4096, 256 rows a group 167 + 16 =
// 0.42 PFLOP/s, matrix units busy for a third and vector units for half of it).
#pragma once

#include "tp_ops_common.h"

#include <algorithm>
#include <type_traits>

namespace tp {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));

// Where a running maximum starts: finite, so that a score of -infinity has
// probability e^-inf = 0 and not NaN, also where every score is -infinity.
constexpr float kLeastScore = -3.0e38f;
constexpr int kTile = 32;      // tokens of a wave's step
constexpr int kRowTile = 16;  // query rows: columns of a matrix instruction

// Waves of a workgroup; a unit is a step of each.  One workgroup per CU: 64 KB of
// loads in flight keep it busy (4 waves of 64 columns have half, 8 the same).
// More only add starts and joins: 64 x 8192 tokens, 8 heads of 128, 4 waves, 1 / 2
// / 3 workgroups per CU 354 / 392 / 362 us, 1 x 131072 104 / 117 / 117; 8 waves
// 357 and 107, and 12.3 us for 1 x 577 against 9.7 (fewer, longer units).
template <int DP, int H>
__host__ __device__ constexpr int paged_waves() {
  return DP <= 64 && H == 1 ? 8 : 4;
}

template <int DP, int H>
__host__ __device__ constexpr int paged_threads() {
  return 64 * (H > 1 ? 2 : 1) * paged_waves<DP, H>();
}

struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  const int32_t *block_table, *lengths;
  float* parts;        // two states per workgroup
  uint32_t* counters;  // per (sequence, cache head, row group): states left so far; zero between launches
  const int64_t* ancestors;  // of new tokens (NULL: a chain)
  int64_t q_batch, q_token, q_head, kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  int64_t n_pages, table_width, window, sinks;
  int batch, tokens, hq, hkv, group, row_groups, d, page_size;
  float scale;  // of the scores, in base 2
};

// The row that masked tokens' loads read, and masked columns'.
__device__ const uint4 kZeros[32] = {};

// A 16-byte load from global memory (said so: of a pointer chosen from two, the
// compiler would make a flat load, whose wait covers LDS too).  ONCE: past the caches.
template <bool ONCE, typename V>
__device__ __forceinline__ V load16(const void* p) {
  const auto at = (const __attribute__((address_space(1))) V*)p;
  return ONCE ? __builtin_nontemporal_load(at) : *at;
}

// kUnit: of the probabilities, the sums and the outputs of a state (a power of
// two, which the last division takes out).  In fp16 the largest is 2^15, so that
// those down to 2^-39 of it count (of a largest of 1 those below 2^-25 would be
// in the sum alone); bf16 has the exponents of fp32.
//
// cut: a probability as two numbers of T, its leading bits and what they leave,
// for a product each: 2^-16 (bf16) or 2^-22 of it are lost, where one number
// loses 2^-9 or 2^-12, and its error is as large as the output's rounding.  The
// second products run under the loads (64 x 8192 tokens 351 us with and without,
// 1 x 577 9.1 and 9.2).  What a probability above 0 leaves is not 0 (a unit that
// the sum does not feel): 0 times a value that is infinite would be NaN.
//
// cut_above: the same where the leading bits are those of a little less, so that
// what they leave is above 0 by itself (2^-16 or 2^-21 of it are lost).
template <typename T>
struct Mma;
template <>
struct Mma<f16_t> {
  typedef f16x8 v8;
  static constexpr float kUnit = 0x1p15f;
  static constexpr uint32_t kExponent = 0x7c00;  // (all ones: not finite)
  __device__ __forceinline__ static void cut(float x, float y, v8& p, v8& rest, int e) {
    const auto lead = __builtin_amdgcn_cvt_pkrtz(x, y);
    p[e] = (f16_t)lead[0], p[e + 1] = (f16_t)lead[1];
    rest[e] = (f16_t)fmaxf(x - (float)lead[0], fminf(x, 0x1p-24f));
    rest[e + 1] = (f16_t)fmaxf(y - (float)lead[1], fminf(y, 0x1p-24f));
  }
  __device__ __forceinline__ static void cut_above(float x, float y, v8& p, v8& rest, int e) {
    const auto lead = __builtin_amdgcn_cvt_pkrtz(x * (1.0f - 0x1p-11f), y * (1.0f - 0x1p-11f));
    p[e] = (f16_t)lead[0], p[e + 1] = (f16_t)lead[1];
    rest[e] = (f16_t)(x - (float)lead[0]), rest[e + 1] = (f16_t)(y - (float)lead[1]);
  }
  __device__ __forceinline__ static f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<bf16_t> {
  typedef bf16x8 v8;
  static constexpr float kUnit = 1.0f;
  static constexpr uint32_t kExponent = 0x7f80;
  __device__ __forceinline__ static void cut(float x, float y, v8& p, v8& rest, int e) {
    const uint32_t xb = __builtin_bit_cast(uint32_t, x), yb = __builtin_bit_cast(uint32_t, y);
    const uint32_t lead = __builtin_amdgcn_perm(yb, xb, 0x07060302);  // their upper halves
    const auto both = __builtin_bit_cast(bf16x2, lead);
    p[e] = both[0], p[e + 1] = both[1];
    rest[e] = (bf16_t)fmaxf(x - __builtin_bit_cast(float, xb & 0xffff0000u), fminf(x, 0x1p-100f));
    rest[e + 1] = (bf16_t)fmaxf(y - __builtin_bit_cast(float, yb & 0xffff0000u), fminf(y, 0x1p-100f));
  }
  __device__ __forceinline__ static void cut_above(float x, float y, v8& p, v8& rest, int e) {
    const uint32_t xb = __builtin_bit_cast(uint32_t, x * (1.0f - 0x1p-8f)), yb = __builtin_bit_cast(uint32_t, y * (1.0f - 0x1p-8f));
    const auto both = __builtin_bit_cast(bf16x2, __builtin_amdgcn_perm(yb, xb, 0x07060302));
    p[e] = both[0], p[e + 1] = both[1];
    rest[e] = (bf16_t)(x - __builtin_bit_cast(float, xb & 0xffff0000u));
    rest[e + 1] = (bf16_t)(y - __builtin_bit_cast(float, yb & 0xffff0000u));
  }
  __device__ __forceinline__ static f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// TREE: exponents above the largest that they are about, at most, and the unit's
// exponent: fp16 probabilities go up to 2^15 (those down to 2^-35 of that largest
// count).
constexpr float kSlack = 4.0f;
template <typename T>
constexpr float kTreeUnit = __is_same(T, f16_t) ? 11.0f : 0.0f;

// Exponents are one fma(score, scale, unit - m).  m is a rounded product, so that the
// largest's is off from its unit by up to m's last bit: by an eighth at kFar, which every
// probability of a row shares and the division takes out, and past that by more than the
// types hold (scores of 2^27: fp16 probabilities of 2^19).  There the product is rounded
// first, as m is, and m is taken from it.
constexpr float kFar = 0x1p20f;

// a b by itself, never a part of an fma.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  const float p = a * b;
  return p;
}

// Floats of a state: per row its maximum and sum, then the (unnormalised) outputs.
template <int DP, int RT>
__host__ __device__ constexpr int state_floats() {
  return RT * kRowTile * (DP + 2);
}

// Addresses of a token's rows in the caches; kZeros: masked.
struct TokenRows {
  uint64_t k, v;
};

// TREE: the new tokens that a row sees, and where its window begins.
struct RowSight {
  uint64_t bits;
  int first, unused;
};

// (13 new tokens of 32 sequences of 0 to 8191 tokens, 8 cache heads of 128: 0 / 1 / 2
// / 3 / 4 / 6 units 207 / 163 / 150 / 141 / 146 / 147 us, of 61 such 401 / 319 / 289 /
// 294 / 291 / 290; 32 of 4096 tokens each 126 / 129 / 128 / 131 / 129 / 130.  256 rows,
// whose units take longer: 64 new tokens of 16 sequences of 0 to 8191, 0 / 1 / 2 / 3 / 4
// units 280 / 183 / 164 / 157 / 166 us, of 16 of 4096 each 157 / 155 / 163 / 163 / 169.
// Of 64 rows 3 and 4 are alike: what 4 loses of the 32 sequences it gains on the 61 and
// on the even ones.  Of 256 rows 3 is best for uneven sequences and costs even ones 6 us.)
template <int H>
constexpr int kLead = H == 1 ? 0 : H == 2 ? 4 : 3;

// Tokens of a sequence that attention reads: [0, sinks) and [first, len).  They
// are counted through in tiles from 0: the first `near` of the count are the
// tokens themselves, those behind lie `shift` further on.
//
// TREE: of any of the new tokens; `before` are in the cache before those.
struct Span {
  int first, len, sinks, near, shift, units, before;
  __device__ __forceinline__ int token(int at) const { return at + (at < near ? 0 : shift); }
};

// LEAD: units without tokens that a (sequence, cache head, row group) begins with, for
// what its beginning and end cost: a workgroup of several short ones takes fewer tokens.
template <int UNIT, bool TREE, int LEAD>
__device__ __forceinline__ Span span_of(const PagedArgs& a, int length) {
  Span s;
  // (room for the last unit's tokens below 2^31)
  if constexpr (TREE) {
    s.before = min(max(length, 0), 0x7fffe000);
    s.len = (int)min((int64_t)(s.before + a.tokens), a.table_width * a.page_size);
    // (a new token without ancestors is at the last one before it)
    s.first = a.window > 0 && s.before > a.window ? (int)(s.before - a.window) : 0;
    s.first = min(s.first, s.len);
  } else {
    s.len = s.before = (int)min(min((int64_t)max(length, 0), a.table_width * a.page_size), (int64_t)0x7ffff000);
    s.first = a.window > 0 && s.len > a.window ? (int)(s.len - a.window) : 0;
  }
  const int base = s.first & ~(kTile - 1);
  s.sinks = (int)min(a.sinks, (int64_t)s.first);
  s.near = (s.sinks + kTile - 1) & ~(kTile - 1);
  s.shift = max(base - s.near, 0);  // (sinks up to the window's own tiles: nothing lies between)
  // (an empty sequence is one unit too: its zeros have to be written)
  s.units = LEAD + max(1, (s.len - s.shift + UNIT - 1) / UNIT);
  return s;
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int64_t u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

__device__ __forceinline__ int opaque(int v) {
  __asm__ volatile("" : "+v"(v));
  return v;
}

// A value that all lanes share, where the compiler cannot see that they do.
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The first `states` waves' states joined: f(row, column, 4 outputs, maximum, sum) for each
// of `rows` rows, row_of(0) and on, below `end` and 4 columns.  Wave w's outputs of the j-th
// are DP floats at `at(w, j)`, its maxima and sums ml[0][w] and ml[1][w].
template <int DP, int W, int R, int THREADS, typename A, typename O, typename F>
__device__ __forceinline__ void join_waves(int tid, int rows, int end, int states, const float (&ml)[2][W][R], A at, O row_of, F f) {
  for (int i = tid; i < rows * (DP / 4); i += THREADS) {
    const int j = i / (DP / 4), c = 4 * (i - j * (DP / 4)), h = row_of(j);
    if (h >= end) continue;
    float top = kLeastScore;
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (w < states) top = MaxOp::of(top, ml[0][w][h]);
    float sum = 0.0f;
    f32x4 y{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (w < states) {
        const float e = __builtin_amdgcn_exp2f(ml[0][w][h] - top);
        sum += e * ml[1][w][h];
        y += e * *reinterpret_cast<const f32x4*>(at(w, j) + c);
      }
    f(h, c, y, top, sum);
  }
}

template <typename T>
__device__ __forceinline__ void store_out(T* out, int d, int c, f32x4 y, float sum) {
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (nothing seen: zeros)
  if (c >= d) return;
  struct {
    T v[4];
  } r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.v[e] = (T)(y[e] * inv);
  __builtin_memcpy(out + c, &r, sizeof(r));
}

// Two floats (8-byte aligned) stored to, or loaded from, where every XCD sees them.
__device__ __forceinline__ void put_device(float* p, float x, float y) {
  const uint64_t v = (uint64_t)__builtin_bit_cast(uint32_t, y) << 32 | __builtin_bit_cast(uint32_t, x);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 get_device(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return f32x2{__builtin_bit_cast(float, (uint32_t)v), __builtin_bit_cast(float, (uint32_t)(v >> 32))};
}

// H RT tiles of 16 query rows share the keys and values that a workgroup reads.  H > 1:
// of its eight waves four load keys and four values, past LDS for all; H sets of 8 / H
// waves each take RT tiles of rows, and the waves of a set every (8 / H)-th of the four
// tiles of tokens.  (Two waves on a SIMD, one of whose matrix instructions run under the
// other's exponentials: 16 new tokens over 131072 170 us with one wave of 64 rows.)  A
// row is a query head of the cache head; TREE: row r is new token r / group's head r %
// group.
template <typename T, int DP, bool EXACT, int RT, int H, bool TREE>
__global__ void __launch_bounds__((paged_threads<DP, H>()), 1) paged_attention_kernel(const PagedArgs a) {
  constexpr int W = paged_waves<DP, H>(), UNIT = W * kTile, MINE = RT * kRowTile, ROWS = H * MINE;
  constexpr int THREADS = paged_threads<DP, H>(), WAVES = THREADS / 64, G = WAVES / H;  // G: waves of a set
  typedef typename Mma<T>::v8 v8;
  typedef int16_t i16x8 __attribute__((ext_vector_type(8)));
  constexpr int LEAD = kLead<H>;
  constexpr int KS = DP / 32;        // k steps of S^T
  constexpr int DT = DP / 16;        // row tiles of O^T
  constexpr int C = DP / 8;          // 16-byte chunks of a row
  constexpr int VL = C / 2;          // V loads per lane and tile
  constexpr int kRow = 2 * DP + 32;  // LDS bytes of a V row: 16 rows' 32-byte pieces fall on distinct banks
  // H > 1: rows of keys lie 16 bytes further apart in LDS than they are long, so that 16
  // rows' pieces are on distinct banks.
  constexpr bool SHARED = H > 1;
  constexpr int kRowK = 2 * DP + 16;
  // a wave's values (or keys), then its outputs of a tile of rows
  constexpr int kPiece = kTile * kRow;
  static_assert(kPiece >= kTile * kRowK && kPiece >= kRowTile * DP * 4 && (H > 1 || W * kPiece >= ROWS * DP * 4), "");
  __shared__ __attribute__((aligned(16))) char v_lds[WAVES][kPiece];
  __shared__ TokenRows rows[WAVES][2][kTile];
  __shared__ float ml[2][G][ROWS];
  __shared__ uint32_t ticket;
  __shared__ RowSight sight[TREE ? WAVES : 1][TREE ? MINE : 1];  // (a wave's own copy: read where a tile is hidden from some)
  // TREE: outputs that are +infinity (1), -infinity (2) or NaN (3) by a value that is,
  // 16 in a word; whether there are any.
  __shared__ uint32_t odd_out[TREE ? ROWS : 1][TREE ? DP / 16 : 1], odd_any;
  if constexpr (TREE) {
    for (int x = threadIdx.x; x < ROWS * (DP / 16); x += THREADS) odd_out[x / (DP / 16)][x % (DP / 16)] = 0;
    if (threadIdx.x == 0) odd_any = 0;
    __syncthreads();
  }
  // Many rows' queries are read from LDS at each tile, in the order of the operands:
  // registers hold no more beside the outputs.  (256 rows' would fill it.)
  constexpr bool Q_LDS = H * RT > 1 && H <= 2;
  // 256 columns: the next keys' registers are free only behind the values' products.
  constexpr bool K_LATE = RT > 1 && DP > 192;
  __shared__ __attribute__((aligned(16))) v8 q_lds[Q_LDS ? H * RT : 1][KS][64];

  const int lane0 = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = SHARED ? wave / W : 0, first_tile = wave - half * W;  // of keys or values, its tile of each W to load
  const int set = SHARED ? wave / G : 0, first_seen = wave - set * G;    // its rows, and its first tile of each W
  const int per_seq = a.hkv * a.row_groups;  // (cache head, row group) pairs of a sequence
  const int all_rows = TREE ? a.tokens * a.group : a.group;

  // All units, and this workgroup's run of them.
  const int units0 = span_of<UNIT, TREE, LEAD>(a, lane0 < a.batch ? a.lengths[lane0] : 0).units;
  auto units_of = [&](int b0) __attribute__((always_inline)) {
    const int x = b0 + lane0;
    const int u = b0 == 0 ? units0 : span_of<UNIT, TREE, LEAD>(a, x < a.batch ? a.lengths[x] : 0).units;
    return x < a.batch ? (int64_t)u * per_seq : (int64_t)0;
  };
  const int64_t upto0 = wave_scan(units_of(0), lane0);  // inclusive, of the first 64 sequences
  int64_t total = __shfl(upto0, 63);
  for (int b0 = 64; b0 < a.batch; b0 += 64) total += __shfl(wave_scan(units_of(b0), lane0), 63);
  total = uniform(total);
  // (no more workgroups than units: every run holds one at least)
  const int64_t wgs = min((int64_t)gridDim.x, total);
  if (blockIdx.x >= wgs) return;
  int64_t at = blockIdx.x * total / wgs;
  const int64_t start = at, end = (blockIdx.x + 1) * total / wgs;
  // the sequence of its first unit
  int b = 0;
  int64_t seq0 = 0;  // units before sequence b
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int64_t u = units_of(b0), upto = b0 == 0 ? upto0 : wave_scan(u, lane0) + seq0;
    const uint64_t above = __ballot(b0 + lane0 < a.batch && upto > at);
    if (above) {
      const int l = __builtin_ctzll(above);
      b = b0 + l;
      seq0 = __shfl(upto - u, l);
      break;
    }
    seq0 = __shfl(upto, 63);
  }
  b = __builtin_amdgcn_readfirstlane(b);
  seq0 = uniform(seq0);
  Span sp = span_of<UNIT, TREE, LEAD>(a, a.lengths[b]);

  const int sinks = (int)min(a.sinks, (int64_t)0x7fffffff);
  // TREE: scores are scaled behind their maximum, so a negative scale's sign goes
  // to the queries (and a scale of 0 is next to it: 0 times a masked -infinity).
  const float scale = TREE ? fmaxf(fabsf(a.scale), 1e-30f) : a.scale;
  const uint32_t q_sign = TREE && a.scale < 0.0f ? 0x80008000u : 0u;
  auto signed_q = [&](v8 q) __attribute__((always_inline)) {
    return TREE ? __builtin_bit_cast(v8, __builtin_bit_cast(u32x4, q) ^ q_sign) : q;
  };

  while (at < end) {
    // a segment: units [j0, j1) of one (sequence, cache head, row group)
    // (opaque per segment: addresses made from it are not kept across segments,
    // nor those of the join across the tiles)
    const int lane = opaque(lane0), lr = lane & 15, lg = lane >> 4;
    const int64_t off = at - seq0;
    const int pair = (int)(off / sp.units);
    const int j0 = (int)(off - (int64_t)pair * sp.units);
    const int j1 = (int)min((int64_t)sp.units, j0 + (end - at));
    const int kvh = pair / a.row_groups, rg = pair - kvh * a.row_groups;
    const int row0 = rg * ROWS;  // first query row
    const int heads = min(ROWS, all_rows - row0);
    const int32_t* bt = a.block_table + (int64_t)b * a.table_width;
    const T* kbase = static_cast<const T*>(a.k) + kvh * a.kc_head;
    const T* vbase = static_cast<const T*>(a.v) + kvh * a.vc_head;
    const T* zeros = reinterpret_cast<const T*>(kZeros);
    const T* mine_base = half == 0 ? kbase : vbase;  // SHARED
    const int64_t mine_page = half == 0 ? a.kc_page : a.vc_page, mine_slot = half == 0 ? a.kc_slot : a.vc_slot;

    const int unit0 = LEAD ? max(j0 - LEAD, 0) : j0;  // first of tokens
    const int tiles = (LEAD ? max(j1 - LEAD, 0) - unit0 : j1 - j0) * W;
    auto first_of = [&](int i) __attribute__((always_inline)) { return sp.token(unit0 * UNIT + i * kTile); };  // token of tile i
    auto page_of = [&](int i) __attribute__((always_inline)) {  // of lane's token of tile i; -1: masked
      const int t = first_of(i) + (lane & 31);
      int page = -1;
      if (i < tiles && (t >= sp.first || t < sp.sinks) && t < sp.len) page = bt[(uint32_t)t / (uint32_t)a.page_size];
      return page;  // (looked at by put_rows, a step later: here it would be waited for)
    };
    int page0 = -1, page = -1;  // TREE: ahead of the queries and their sights
    if constexpr (TREE) page0 = page_of(first_tile), page = page_of(first_tile + W);

    // Q^T: a lane holds columns 32 s + 8 lg .. + 7 of row 16 r + lr
    v8 q[Q_LDS ? 1 : RT][KS];
    int all_first = 0;  // TREE: where the last row's window begins
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = row0 + set * MINE + kRowTile * r + lr;
      const T* p = static_cast<const T*>(a.q) + b * a.q_batch;
      if constexpr (TREE) {
        const int token = min(row, all_rows - 1) / a.group;
        p += token * a.q_token + (kvh * a.group + row - token * a.group) * a.q_head;
        const uint64_t all = ~0ull >> (64 - a.tokens);
        uint64_t bits = (a.ancestors ? (uint64_t)a.ancestors[(int64_t)b * a.tokens + token] : ~0ull >> (63 - token)) & all;
        int first = 0;
        if (a.window > 0) {
          const int depth = __builtin_popcountll(bits);
          first = (int)max((int64_t)sp.before + depth - a.window, (int64_t)0);
          // a window ends among the new tokens (one whose entry is 0 is at the last place before them)
          if (__any(depth >= a.window)) {
            const int64_t here = (int64_t)sp.before - 1 + depth;
            for (int j = 0; j < a.tokens; ++j) {
              const uint64_t other = (a.ancestors ? (uint64_t)a.ancestors[(int64_t)b * a.tokens + j] : ~0ull >> (63 - j)) & all;
              const int64_t place = (int64_t)sp.before - 1 + __builtin_popcountll(other);
              if (place <= here - a.window && place >= a.sinks) bits &= ~(1ull << j);
            }
          }
          all_first = max(all_first, first);
        }
        if (lane < kRowTile) sight[wave][kRowTile * r + lane] = RowSight{bits, first, 0};
      } else {
        p += (kvh * a.group + row) * a.q_head;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bool in = row - row0 < heads && (EXACT || 32 * s + 8 * lg < a.d);
        if constexpr (!Q_LDS) q[r][s] = signed_q(load16<!TREE, v8>(in ? p + 32 * s + 8 * lg : zeros));
        else if (first_seen == (r * KS + s) % G) q_lds[set * RT + r][s][lane] = signed_q(load16<!TREE, v8>(in ? p + 32 * s + 8 * lg : zeros));
      }
    }
    if constexpr (TREE) {
      if (a.window > 0) {
#pragma unroll
        for (int o = 1; o < 16; o *= 2) all_first = max(all_first, __shfl_xor(all_first, o));
        all_first = __builtin_amdgcn_readfirstlane(all_first);
      }
    }

    if constexpr (Q_LDS || SHARED) __syncthreads();

    auto put_rows = [&](int i, int page) __attribute__((always_inline)) {
      const int t = first_of(i) + (lane & 31);
      const uint32_t slot = (uint32_t)t % (uint32_t)a.page_size;
      TokenRows r{(uint64_t)zeros, (uint64_t)zeros};
      if constexpr (SHARED) {  // (a wave loads keys or values: .k is its own row)
        if (page >= 0 && page < a.n_pages) r.k = (uint64_t)(mine_base + page * mine_page + slot * mine_slot);
        if (lane < kTile) rows[wave][(i / W) & 1][lane].k = r.k;
        return;
      }
      if (page >= 0 && page < a.n_pages)
        r = TokenRows{(uint64_t)(kbase + page * a.kc_page + slot * a.kc_slot), (uint64_t)(vbase + page * a.vc_page + slot * a.vc_slot)};
      if (lane < kTile) rows[wave][(i / W) & 1][lane] = r;
    };
    v8 k[SHARED ? 1 : 2][KS], v[VL];
    auto load_k = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const T* r = reinterpret_cast<const T*>(rows[wave][(i / W) & 1][16 * h + lr].k) + 8 * lg;
#pragma unroll
        for (int s = 0; s < KS; ++s) k[h][s] = load16<!TREE, v8>(EXACT || 32 * s + 8 * lg < a.d ? r + 32 * s : zeros);
      }
    };
    // chunk c of a lane: 16-byte piece v_piece(c) of token v_token(c)
    auto v_token = [&](int c) __attribute__((always_inline)) { return 64 % C == 0 ? lane / C + c * (64 / C) : (lane + 64 * c) / C; };
    auto v_piece = [&](int c) __attribute__((always_inline)) { return 64 % C == 0 ? lane % C : (lane + 64 * c) % C; };
    auto load_v = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < VL; ++c) {
        const TokenRows& at = rows[wave][(i / W) & 1][v_token(c)];
        const T* r = reinterpret_cast<const T*>(SHARED ? at.k : at.v) + 8 * v_piece(c);
        v[c] = load16<!TREE, v8>(EXACT || 8 * v_piece(c) < a.d ? r : zeros);
      }
    };

    f32x4 o[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int t = 0; t < DT; ++t) o[r][t] = f32x4{0, 0, 0, 0};
      m[r] = kLeastScore, l[r] = 0.0f;
    }

    put_rows(first_tile, TREE ? page0 : page_of(first_tile));
    wave_lds_fence();
    // (in the loop's order, next pages, keys, values: its waits count loads)
    if constexpr (!TREE) page = page_of(first_tile + W);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!SHARED) {
      load_k(first_tile);
      __builtin_amdgcn_sched_barrier(0);
    }
    load_v(first_tile);
    __builtin_amdgcn_sched_barrier(0);
    auto put_v = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < VL; ++c) *reinterpret_cast<v8*>(v_lds[wave] + v_token(c) * kRow + 16 * v_piece(c)) = v[c];
    };
    // TREE: a value that is not finite may meet only the rows that see it.  In tiles
    // that are hidden from some it is noted for those that do, and zero in LDS.
    auto clean_v = [&](int i) __attribute__((always_inline)) {
      const int t0 = first_of(i);
      if (t0 + kTile <= sp.before && (a.window <= 0 || t0 >= sp.before + a.tokens - a.window || t0 + kTile <= a.sinks)) return;
      // two values a word: a half of what an exponent lacks is 0 where it is all ones,
      // else it carries into the half's top bit
      uint32_t finite = ~0u;
#pragma unroll
      for (int c = 0; c < VL; ++c) {
        const u32x4 w = __builtin_bit_cast(u32x4, v[c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) finite &= (~w[e] & Mma<T>::kExponent * 0x10001u) + 0x7fff7fffu;
      }
      if (!__any((finite & 0x80008000u) != 0x80008000u)) return;
      wave_lds_fence();
#pragma unroll 1
      for (int c = lane; c < kTile * DP; c += 64) {
        T* at = reinterpret_cast<T*>(v_lds[wave] + c / DP * kRow) + c % DP;
        const uint32_t w = __builtin_bit_cast(uint16_t, *at);
        if ((w & Mma<T>::kExponent) != Mma<T>::kExponent) continue;
        *at = (T)0.0f;
        const uint32_t is = w & (0x7fff & ~Mma<T>::kExponent) ? 3 : w >> 15 ? 2 : 1;
        const int t = t0 + c / DP, j = t - sp.before;
#pragma unroll 1
        for (int r = 0; r < ROWS; ++r) {
          const RowSight mine = sight[H == 1 ? wave : r / MINE * G][r % MINE];
          if (j < 0 ? t >= mine.first || t < a.sinks : j < a.tokens && (mine.bits >> (j & 63) & 1))
            atomicOr(&odd_out[r][c % DP / 16], is << (2 * (c % 16)));
        }
      }
      if (lane == 0) odd_any = 1;
      wave_lds_fence();
    };
    // V^T: a lane takes column 16 t + lr of tokens 16 h + 4 lg .. + 3
    auto read_v = [&](int v_wave, int t) __attribute__((always_inline)) {  // (whose piece holds the values)
      i16x4 part[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4*)(v_lds[v_wave] + (16 * h + 4 * lg + (lr >> 2)) * kRow + 32 * t +
                                                       8 * (lr & 3)));
      return (i16x8)__builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    };
    if constexpr (!TREE) {
      for (int i = first_tile; i < tiles; i += W) {
        // rows of the next tile, pages of the one after
        const uint64_t masked = __ballot(rows[wave][(i / W) & 1][lane & 31].k == (uint64_t)zeros);
        put_rows(i + W, page);
        wave_lds_fence();
        page = page_of(i + 2 * W);

        f32x4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          s[h] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < KS; ++c) s[h] = Mma<T>::mul(k[h][c], q[0][c], s[h]);
        }
        // (sched_barrier: moved up, the loads would take registers of their own)
        __builtin_amdgcn_sched_barrier(0);
        load_k(i + W);

        // lane: row lr, tokens 16 h + 4 lg + e
#pragma unroll
        for (int h = 0; h < 2; ++h) s[h] *= a.scale;
        if (masked) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (masked >> (16 * h + 4 * lg + e) & 1) s[h][e] = -INFINITY;
        }
        float top = m[0];  // (a NaN is not its maximum, but makes its exponential, so the sums, NaN)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, s[h][e]);
        top = combine32<MaxOp>(combine16<MaxOp>(top));
        const float keep = __builtin_amdgcn_exp2f(m[0] - top);
        m[0] = top;
        l[0] *= keep;
        float x8[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = __builtin_amdgcn_exp2f(s[h][e] - top) * Mma<T>::kUnit;
            l[0] += x;
            x8[4 * h + e] = x;
          }
        v8 p, rest;
#pragma unroll
        for (int e = 0; e < 8; e += 2) Mma<T>::cut(x8[e], x8[e + 1], p, rest, e);
#pragma unroll
        for (int t = 0; t < DT; ++t) o[0][t] *= keep;

        put_v();
        wave_lds_fence();
        __builtin_amdgcn_sched_barrier(0);
        load_v(i + W);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const v8 both = __builtin_bit_cast(v8, read_v(wave, t));
          o[0][t] = Mma<T>::mul(both, p, o[0][t]);
          o[0][t] = Mma<T>::mul(both, rest, o[0][t]);
          if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (eight reads at a time: registers)
        }
        wave_lds_fence();
      }
    } else {
      // The largest that exponents are about is moved only where one is above it by
      // more than kSlack, outside the loop over the tiles: within, the outputs are
      // the matrix instructions' alone and stay in their registers (64 rows of 128
      // columns: 128 products and 400 copies a tile otherwise).
      int i = first_tile;
      bool fresh = true;    // nothing is summed yet: there is nothing to scale
      bool far = false;     // of some row of the wave |m| is above kFar
      auto is_far = [&]() __attribute__((always_inline)) {
        bool is = false;
#pragma unroll
        for (int r = 0; r < RT; ++r) is |= fabsf(m[r]) > kFar && m[r] > kLeastScore;
        return __any(is) != 0;
      };
      bool staged = false;  // SHARED: W tiles are in LDS, of which a wave takes every G-th
      int seen = first_seen, step = W;
      while (i < tiles) {
        float top[RT];
        bool above = false;
        for (; i < tiles; i += G < W ? step : W) {
          if constexpr (SHARED) {
            if (!staged) {
              // this tile past LDS, the next one's loads behind it
              if (half == 0) {
#pragma unroll
                for (int c = 0; c < VL; ++c) *reinterpret_cast<v8*>(v_lds[wave] + v_token(c) * kRowK + 16 * v_piece(c)) = v[c];
              } else {
                put_v();
                clean_v(i);
              }
              __syncthreads();
              put_rows(i + W, page);
              wave_lds_fence();
              page = page_of(i + 2 * W);
              __builtin_amdgcn_sched_barrier(0);
              load_v(i + W);
              __builtin_amdgcn_sched_barrier(0);
            }
            staged = true;
          }
          const int piece = !SHARED ? wave : G == W ? first_seen : seen, tile = SHARED ? i - first_tile + piece : i;
          f32x4 s[RT][2];
          v8 kc[2][KS];
          const bool mine_masked = rows[piece][(i / W) & 1][lane & 31].k == (uint64_t)zeros;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < KS; ++c)
              kc[h][c] = SHARED ? *reinterpret_cast<const v8*>(v_lds[piece] + (16 * h + lr) * kRowK + 64 * c + 16 * lg) : k[SHARED ? 0 : h][c];
          if constexpr (SHARED) __builtin_amdgcn_sched_barrier(0);  // (all reads from LDS in flight)
#pragma unroll
          for (int c = 0; c < KS; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                if (c == 0) s[r][h] = f32x4{0, 0, 0, 0};
                s[r][h] = Mma<T>::mul(kc[h][c], Q_LDS ? q_lds[set * RT + r][c][lane] : q[r][c], s[r][h]);
              }
          // lane: row 16 r + lr, tokens 16 h + 4 lg + e
          const uint64_t masked = __ballot(mine_masked);
          if (masked) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (masked >> (16 * h + 4 * lg + e) & 1) {
#pragma unroll
                  for (int r = 0; r < RT; ++r) s[r][h][e] = -INFINITY;
                }
          }
          // tokens that some rows see and others do not
          const int t0 = first_of(tile);
          const bool some = !(t0 + kTile <= sp.before && (t0 >= all_first || t0 + kTile <= a.sinks));
          if (some) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const RowSight mine = sight[wave][kRowTile * r + lr];
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  // (no short cuts: as branches they are 8 RT small blocks, run once or twice a segment)
                  const int t = t0 + 16 * h + 4 * lg + e, j = t - sp.before;
                  const int cached = (int)(t >= mine.first) | (int)(t < sinks);
                  const int drafted = (int)(mine.bits >> (j & 63)) & (int)(j < a.tokens);
                  s[r][h][e] = (j < 0 ? cached : drafted) & 1 ? s[r][h][e] : -INFINITY;
                }
            }
          }
          above = false;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            top[r] = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e) top[r] = fmaxf(top[r], s[r][h][e]);
            top[r] = product(combine32<MaxOp>(combine16<MaxOp>(top[r])), scale);
            above |= top[r] - m[r] > kSlack;
          }
          if (__any(above)) {
            if (!fresh) {  // (the tile is begun again)
              above = true;
              break;
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) m[r] = top[r] - m[r] > kSlack ? top[r] : m[r];
            far = is_far();
          }
          above = fresh = false;
          if constexpr (!SHARED) {
            // rows of the next tile, pages of the one after
            put_rows(i + W, page);
            wave_lds_fence();
            page = page_of(i + 2 * W);
            __builtin_amdgcn_sched_barrier(0);
            if (!K_LATE) load_k(i + W);
          }

          // values are read from LDS two tiles of columns ahead of their products, the
          // first ones ahead of the exponentials
          v8 both[2][2];
          auto read_two = [&](int t) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 2; ++u) both[t / 2 & 1][u] = __builtin_bit_cast(v8, read_v(SHARED ? W + piece : wave, t + u));
          };
          if constexpr (SHARED) {
            read_two(0);
            __builtin_amdgcn_sched_barrier(0);
          }

          if (far) {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[r][h][e] = product(s[r][h][e], scale) - m[r];
          }
          const float each = far ? 1.0f : scale;

          v8 p[RT], rest[RT];
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const float about = kTreeUnit<T> - (far ? 0.0f : m[r]);
            float x8[8];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][h][e], each, about));
                l[r] += x;
                x8[4 * h + e] = x;
              }
#pragma unroll
            for (int e = 0; e < 8; e += 2) Mma<T>::cut_above(x8[e], x8[e + 1], p[r], rest[r], e);
          }
          // a value that is not finite may meet only the rows that see it
          if constexpr (!SHARED) {
            put_v();
            clean_v(i);
            wave_lds_fence();
            __builtin_amdgcn_sched_barrier(0);
            load_v(i + W);
            __builtin_amdgcn_sched_barrier(0);
            read_two(0);
          }
#pragma unroll
          for (int t = 0; t < DT; t += 2) {
            if (t + 2 < DT) read_two(t + 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int r = 0; r < RT; ++r) o[r][t + u] = Mma<T>::mul(both[t / 2 & 1][u], p[r], o[r][t + u]);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int r = 0; r < RT; ++r) o[r][t + u] = Mma<T>::mul(both[t / 2 & 1][u], rest[r], o[r][t + u]);
            __builtin_amdgcn_sched_barrier(0);
          }
          if constexpr (SHARED) {
            if constexpr (G < W) seen += G, step = 0;
            if (G == W || seen >= W) {
              staged = false;
              if constexpr (G < W) seen = first_seen, step = W;
              __syncthreads();  // (all waves have read the tiles)
            }
          } else {
            wave_lds_fence();
            if (K_LATE) load_k(i + W);
          }
        }
        if (!above) break;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float to = top[r] - m[r] > kSlack ? top[r] : m[r], keep = __builtin_amdgcn_exp2f(m[r] - to);
          m[r] = to;
          l[r] *= keep;
#pragma unroll
          for (int t = 0; t < DT; ++t) o[r][t] *= keep;
        }
        far = is_far();
      }
    }

    // the waves' states, through LDS
    const int tid = opaque((int)threadIdx.x);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      l[r] = combine32<AddOp>(combine16<AddOp>(l[r]));
      if (lane < kRowTile) {
        const int row = set * MINE + kRowTile * r + lane;
        ml[0][first_seen][row] = m[r], ml[1][first_seen][row] = l[r];
      }
    }
    auto with_odd = [&](int h, int c, f32x4 y) __attribute__((always_inline)) {
      if constexpr (TREE) {
        if (odd_any) {
          const uint32_t word = odd_out[h][c / 16] >> (2 * (c % 16));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t is = word >> (2 * e) & 3;
            if (is) y[e] += is == 3 ? __builtin_nanf("") : is == 1 ? INFINITY : -INFINITY;
          }
        }
      }
      return y;
    };
    auto put_out = [&](int h, int c, f32x4 y, float, float sum) __attribute__((always_inline)) {
      int64_t at_row = (int64_t)b * a.hq + kvh * a.group + row0 + h;
      if constexpr (TREE) {
        const int token = (row0 + h) / a.group;
        at_row = ((int64_t)b * a.tokens + token) * a.hq + kvh * a.group + row0 + h - token * a.group;
      }
      store_out(static_cast<T*>(a.out) + at_row * a.d, a.d, c, y, sum);
    };
    // (each set's r-th tile of rows)
    auto join = [&](auto f) __attribute__((always_inline)) {
      float* ow = reinterpret_cast<float*>(v_lds[wave]);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (r > 0) __syncthreads();
#pragma unroll
        for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(ow + lr * DP + 16 * t + 4 * lg) = o[r][t];
        __syncthreads();
        join_waves<DP, G, ROWS, THREADS>(
            tid, H == 1 ? min(kRowTile, heads - kRowTile * r) : H * kRowTile, heads, G, ml,
            [&](int w, int j) __attribute__((always_inline)) {
              return reinterpret_cast<const float*>(v_lds[(H == 1 ? 0 : j / kRowTile * G) + w]) + (H == 1 ? j : j % kRowTile) * DP;
            },
            [&](int j) __attribute__((always_inline)) { return H == 1 ? kRowTile * r + j : j / kRowTile * MINE + kRowTile * r + j % kRowTile; }, f);
      }
    };
    if (j0 == 0 && j1 == sp.units) {
      join([&](int h, int c, f32x4 y, float top, float sum) __attribute__((always_inline)) {
        put_out(h, c, with_odd(h, c, y), top, sum);
      });
    } else {
      // The state goes to the workspace, and the last workgroup of this head
      // joins them all.  They belong to consecutive workgroups g0 .. g1; each
      // but g0 starts its run inside the head (its first segment), and so does
      // g0 if its run starts at unit 0.  States are written and read by
      // device-scope accesses (past the XCDs' own L2s), so that the ticket
      // needs no fence, only the stores' completion: a fence writes back the
      // whole L2 (64 sequences x 8192 tokens of one cache head: 186 us with a
      // fence per workgroup).
      constexpr int STATE = state_floats<DP, H * RT>();
      float* part = a.parts + ((int64_t)blockIdx.x * 2 + (at != start)) * STATE;
      if constexpr (H > 1) {
        // (of many rows a state is 33 KB: another launch joins them on all CUs)
        join([&](int h, int c, f32x4 y, float top, float sum) __attribute__((always_inline)) {
          *reinterpret_cast<f32x4*>(part + 2 * ROWS + h * DP + c) = with_odd(h, c, y);
          if (c == 0) part[2 * h] = top, part[2 * h + 1] = sum;
        });
      } else {
        join([&](int h, int c, f32x4 y, float top, float sum) __attribute__((always_inline)) {
          y = with_odd(h, c, y);
          put_device(part + 2 * ROWS + h * DP + c, y[0], y[1]);
          put_device(part + 2 * ROWS + h * DP + c + 2, y[2], y[3]);
          if (c == 0) put_device(part + 2 * h, top, sum);
        });
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const int64_t u0 = seq0 + (int64_t)pair * sp.units, u1 = u0 + sp.units;
        const int64_t g0 = ((u0 + 1) * wgs - 1) / total, g1 = (u1 * wgs - 1) / total;
        const int n = (int)(g1 - g0 + 1);
        uint32_t* counter = a.counters + (int64_t)b * per_seq + pair;
        if (tid == 0) ticket = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (ticket == (uint32_t)n - 1) {
          if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          const int later = g0 * total / wgs < u0;  // g0's state is its second
          const float* parts = a.parts + (g0 * 2 + later) * STATE;
          const int64_t next = (2 - later) * STATE;  // g0 + 1's, from g0's
          // 64 pieces (a row, 4 columns) of the states are a wave's, or, of few
          // pieces, every PG-th of their states; its loads are in flight together
          const int pieces = heads * (DP / 4), groups = (pieces + 63) / 64, pg = max(1, W / groups);
          float* joined = reinterpret_cast<float*>(v_lds[0]);  // [pg][groups * 64 pieces]
          auto gather = [&](auto ahead) __attribute__((always_inline)) {
            constexpr int A = decltype(ahead)::value;
            for (int x = wave; x < groups * pg; x += WAVES) {
              const int part = x / groups, i = (x - part * groups) * 64 + lane;
              if (i >= pieces) continue;
              const int h = i / (DP / 4), c = 4 * (i - h * (DP / 4));
              float top = kLeastScore, sum = 0.0f;
              f32x4 y{0, 0, 0, 0};
              for (int g = part; g < n; g += pg * A) {
                f32x2 pm[A], po[A][2];
  #pragma unroll
                for (int z = 0; z < A; ++z) {
                  const int gz = min(g + z * pg, n - 1);
                  const float* p = parts + (gz == 0 ? 0 : next + (int64_t)(gz - 1) * 2 * STATE);
                  pm[z] = get_device(p + 2 * h);
                  po[z][0] = get_device(p + 2 * ROWS + h * DP + c);
                  po[z][1] = get_device(p + 2 * ROWS + h * DP + c + 2);
                }
  #pragma unroll
                for (int z = 0; z < A; ++z)
                  if (g + z * pg < n) {
                    const float m2 = MaxOp::of(top, pm[z][0]);
                    const float f = __builtin_amdgcn_exp2f(top - m2), fz = __builtin_amdgcn_exp2f(pm[z][0] - m2);
                    sum = sum * f + pm[z][1] * fz;
                    y = y * f + f32x4{po[z][0][0], po[z][0][1], po[z][1][0], po[z][1][1]} * fz;
                    top = m2;
                  }
              }
              *reinterpret_cast<f32x4*>(joined + part * groups * 256 + h * DP + c) = y;
              if (c == 0) ml[0][part][h] = top, ml[1][part][h] = sum;
            }
          };
          if (n <= 4 * pg) gather(std::integral_constant<int, 4>{});
          else gather(std::integral_constant<int, 16>{});
          __syncthreads();
          join_waves<DP, W, ROWS, THREADS>(
              tid, heads, heads, pg, ml,
              [&](int w, int j) __attribute__((always_inline)) { return joined + w * groups * 256 + j * DP; },
              [&](int j) __attribute__((always_inline)) { return j; }, put_out);
        }
      }
    }
    // (read ahead of the barrier: behind it a wave may note the next segment's)
    bool odd = false;
    if constexpr (TREE) odd = odd_any != 0;
    __syncthreads();
    if constexpr (TREE) {
      if (odd) {  // (the next segment has none yet)
        for (int x = threadIdx.x; x < ROWS * (DP / 16); x += THREADS) odd_out[x / (DP / 16)][x % (DP / 16)] = 0;
        if (threadIdx.x == 0) odd_any = 0;
        __syncthreads();
      }
    }
    at += j1 - j0;
    if (at - seq0 == (int64_t)sp.units * per_seq) {
      seq0 = at;
      if (++b < a.batch) sp = span_of<UNIT, TREE, LEAD>(a, a.lengths[b]);
    }
  }
}

// Rows of a joining workgroup.
template <int RT, int H>
__host__ __device__ constexpr int join_rows() {
  return RT * H > 4 ? 8 : 4;
}

// The states that the tree kernel's workgroups left of a (sequence, cache head, row
// group), joined: blockIdx.x of those, blockIdx.y EACH rows (131072 tokens, 8 cache
// heads of 128 and 64 rows: 4 a workgroup 7.7 us, 16 14).
template <typename T, int DP, int RT, int H>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs a, int grid) {
  constexpr int ROWS = H * RT * kRowTile, EACH = join_rows<RT, H>(), UNIT = paged_waves<DP, H>() * kTile, STATE = ROWS * (DP + 2), A = 8;
  const int lane = threadIdx.x & 63, per_seq = a.hkv * a.row_groups;
  const int b = blockIdx.x / per_seq, pair = blockIdx.x - b * per_seq;
  // units of all sequences, and those before this one
  int64_t total = 0, before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int x = b0 + lane;
    const int64_t u = x < a.batch ? (int64_t)span_of<UNIT, true, kLead<H>>(a, a.lengths[x]).units * per_seq : 0;
    total += __shfl(wave_scan(u, lane), 63);
    before += __shfl(wave_scan(x < b ? u : 0, lane), 63);
  }
  const int units = span_of<UNIT, true, kLead<H>>(a, a.lengths[b]).units;
  const int64_t wgs = min((int64_t)grid, total);
  const int64_t u0 = before + (int64_t)pair * units, u1 = u0 + units;
  const int64_t g0 = ((u0 + 1) * wgs - 1) / total, g1 = (u1 * wgs - 1) / total;
  const int n = (int)(g1 - g0 + 1);
  if (n == 1) return;  // (its outputs are written)
  const int later = g0 * total / wgs < u0;  // g0's state is its second
  const float* parts = a.parts + (g0 * 2 + later) * STATE;
  const int64_t next = (2 - later) * STATE;  // g0 + 1's, from g0's
  const int kvh = pair / a.row_groups, row0 = (pair - kvh * a.row_groups) * ROWS, all_rows = a.tokens * a.group;
  for (int i = threadIdx.x; i < EACH * (DP / 4); i += 128) {
    const int h = blockIdx.y * EACH + i / (DP / 4), c = 4 * (i % (DP / 4));
    if (row0 + h >= all_rows) continue;
    float top = kLeastScore, sum = 0.0f;
    f32x4 y{0, 0, 0, 0};
    for (int g = 0; g < n; g += A) {
      f32x2 pm[A];
      f32x4 po[A];
#pragma unroll
      for (int z = 0; z < A; ++z) {
        const int gz = min(g + z, n - 1);
        const float* p = parts + (gz == 0 ? 0 : next + (int64_t)(gz - 1) * 2 * STATE);
        pm[z] = *reinterpret_cast<const f32x2*>(p + 2 * h);
        po[z] = *reinterpret_cast<const f32x4*>(p + 2 * ROWS + h * DP + c);
      }
#pragma unroll
      for (int z = 0; z < A; ++z)
        if (g + z < n) {
          const float m2 = MaxOp::of(top, pm[z][0]);
          const float f = __builtin_amdgcn_exp2f(top - m2), fz = __builtin_amdgcn_exp2f(pm[z][0] - m2);
          sum = sum * f + pm[z][1] * fz;
          y = y * f + po[z] * fz;
          top = m2;
        }
    }
    const int token = (row0 + h) / a.group;
    const int64_t at_row = ((int64_t)b * a.tokens + token) * a.hq + kvh * a.group + row0 + h - token * a.group;
    store_out(static_cast<T*>(a.out) + at_row * a.d, a.d, c, y, sum);
  }
}

// Columns that the kernel's instance for d holds.
inline int padded_d(int64_t d) { return d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

// Tiles of rows that share a workgroup's keys and values.  256 rows past 128 (calls, 4
// query heads on each of 8 cache heads of 128 columns: 64 new tokens of 16 sequences of
// 4096 tokens 166 us, 64 rows a group 207; 33 of 40 of 500 92 and 118).  Few or short
// sequences, whose lengths only the device knows, lose by it: 33 of one of 30 26 and 20,
// 64 of one of 4096 45 and 32, of 8 of 256 42 and 29.  Wider heads have 32 rows at most,
// each group of which reads the cache again (256 columns: 64 of 16 of 4096 629 us, 16 of
// each 165).
inline int tree_row_tiles(int64_t rows, int dp) {
  return rows <= kRowTile ? 1 : rows <= 2 * kRowTile || dp > 128 ? 2 : rows <= 8 * kRowTile ? 4 : 16;
}

template <typename T, int DP, int RT, int H, bool TREE>
void launch_rows(const PagedArgs& a, hipStream_t s) {
  const dim3 grid((uint32_t)device_cu_count());
  if (a.d == DP) hipLaunchKernelGGL((paged_attention_kernel<T, DP, true, RT, H, TREE>), grid, dim3(paged_threads<DP, H>()), 0, s, a);
  else hipLaunchKernelGGL((paged_attention_kernel<T, DP, false, RT, H, TREE>), grid, dim3(paged_threads<DP, H>()), 0, s, a);
}

// Trees are compiled apart, a type in a file.
int dispatch_tree_f16(const PagedArgs& a, hipStream_t s);
int dispatch_tree_bf16(const PagedArgs& a, hipStream_t s);

template <typename T, int DP, int RT, int H>
void launch_shared(const PagedArgs& a, hipStream_t s) {
  launch_rows<T, DP, RT, H, true>(a, s);
  const dim3 grid((uint32_t)(a.batch * a.hkv * a.row_groups), RT * H * kRowTile / join_rows<RT, H>());
  hipLaunchKernelGGL((paged_join_kernel<T, DP, RT, H>), grid, dim3(128), 0, s, a, device_cu_count());
}

template <typename T, int DP>
void launch_tree(const PagedArgs& a, hipStream_t s) {
  const int tiles = tree_row_tiles((int64_t)a.tokens * a.group, DP);
  if (tiles == 1) return launch_rows<T, DP, 1, 1, true>(a, s);
  if constexpr (DP <= 128) {
    if (tiles == 2) launch_shared<T, DP, 1, 2>(a, s);
    else if (tiles == 4) launch_shared<T, DP, 2, 2>(a, s);
    else launch_shared<T, DP, 2, 8>(a, s);
  } else {
    // (two sets of waves as above take 136 KB of LDS for their tiles, 8 for addresses and
    // 16 for the queries of 32 rows, all that a CU has, beside masks and sums)
    launch_rows<T, DP, 2, 1, true>(a, s);
  }
}

template <typename T>
int dispatch_tree(const PagedArgs& a, hipStream_t s) {
  switch (padded_d(a.d)) {
    case 64: launch_tree<T, 64>(a, s); break;
    case 96: launch_tree<T, 96>(a, s); break;
    case 128: launch_tree<T, 128>(a, s); break;
    case 192: launch_tree<T, 192>(a, s); break;
    default: launch_tree<T, 256>(a, s); break;
  }
  return launch_status();
}

}  // namespace tp
