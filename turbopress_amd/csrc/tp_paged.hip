// Attention of one new token per sequence over a paged cache.  With the running
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
constexpr int kHeadTile = 16;  // query heads of a workgroup: columns of a matrix instruction

// Waves of a workgroup; a unit is a step of each.  One workgroup per CU: 64 KB of
// loads in flight keep it busy (4 waves of 64 columns have half, 8 the same).
// More only add starts and joins: 64 x 8192 tokens, 8 heads of 128, 4 waves, 1 / 2
// / 3 workgroups per CU 354 / 392 / 362 us, 1 x 131072 104 / 117 / 117; 8 waves
// 357 and 107, and 12.3 us for 1 x 577 against 9.7 (fewer, longer units).
template <int DP>
__host__ __device__ constexpr int paged_waves() {
  return DP <= 64 ? 8 : 4;
}

struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  const int32_t *block_table, *lengths;
  float* parts;        // two states per workgroup
  uint32_t* counters;  // per (sequence, head tile): states left so far; zero between launches
  int64_t q_batch, q_head, kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head;
  int64_t n_pages, table_width, window;
  int batch, hq, hkv, group, head_tiles, d, page_size;
  float scale;  // of the scores, in base 2
};

// The row that masked tokens' loads read, and masked columns'.
__device__ const uint4 kZeros[32] = {};

// A 16-byte load from global memory (said so: of a pointer chosen from two, the
// compiler would make a flat load, whose wait covers LDS too).
template <typename V>
__device__ __forceinline__ V load16(const void* p) {
  return __builtin_nontemporal_load((const __attribute__((address_space(1))) V*)p);
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
template <typename T>
struct Mma;
template <>
struct Mma<f16_t> {
  typedef f16x8 v8;
  static constexpr float kUnit = 0x1p15f;
  __device__ __forceinline__ static void cut(float x, float y, v8& p, v8& rest, int e) {
    const auto lead = __builtin_amdgcn_cvt_pkrtz(x, y);
    p[e] = (f16_t)lead[0], p[e + 1] = (f16_t)lead[1];
    rest[e] = (f16_t)fmaxf(x - (float)lead[0], fminf(x, 0x1p-24f));
    rest[e + 1] = (f16_t)fmaxf(y - (float)lead[1], fminf(y, 0x1p-24f));
  }
  __device__ __forceinline__ static f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<bf16_t> {
  typedef bf16x8 v8;
  static constexpr float kUnit = 1.0f;
  __device__ __forceinline__ static void cut(float x, float y, v8& p, v8& rest, int e) {
    const uint32_t xb = __builtin_bit_cast(uint32_t, x), yb = __builtin_bit_cast(uint32_t, y);
    const uint32_t lead = __builtin_amdgcn_perm(yb, xb, 0x07060302);  // their upper halves
    const auto both = __builtin_bit_cast(bf16x2, lead);
    p[e] = both[0], p[e + 1] = both[1];
    rest[e] = (bf16_t)fmaxf(x - __builtin_bit_cast(float, xb & 0xffff0000u), fminf(x, 0x1p-100f));
    rest[e + 1] = (bf16_t)fmaxf(y - __builtin_bit_cast(float, yb & 0xffff0000u), fminf(y, 0x1p-100f));
  }
  __device__ __forceinline__ static f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// Floats of a state: per head its maximum and sum, then the (unnormalised) outputs.
template <int DP>
__host__ __device__ constexpr int state_floats() {
  return kHeadTile * (DP + 2);
}

// Addresses of a token's rows in the caches; kZeros: masked.
struct TokenRows {
  uint64_t k, v;
};

// Tokens of a sequence that attention reads: [first, len); its first unit's base.
struct Span {
  int first, len, base, units;
};

template <int UNIT>
__device__ __forceinline__ Span span_of(const PagedArgs& a, int length) {
  Span s;
  // (room for the last unit's tokens below 2^31)
  s.len = (int)min(min((int64_t)max(length, 0), a.table_width * a.page_size), (int64_t)0x7ffff000);
  s.first = a.window > 0 && s.len > a.window ? (int)(s.len - a.window) : 0;
  s.base = s.first & ~(kTile - 1);
  // (an empty sequence is one unit too: its zeros have to be written)
  s.units = max(1, (s.len - s.base + UNIT - 1) / UNIT);
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

// The first `states` waves' states joined: f(head, column, 4 outputs, maximum, sum) for each
// head and 4 columns.  Wave w's outputs are floats [head][DP] at lds + w * pitch,
// its maxima and sums ml[0][w] and ml[1][w].
template <int DP, int W, typename F>
__device__ __forceinline__ void join_waves(int tid, int heads, int states, const float (&ml)[2][W][kHeadTile],
                                           const char* lds, int pitch, F f) {
  for (int i = tid; i < heads * (DP / 4); i += 64 * W) {
    const int h = i / (DP / 4), c = 4 * (i - h * (DP / 4));
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
        y += e * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * pitch) + h * DP + c);
      }
    f(h, c, y, top, sum);
  }
}

template <typename T>
__device__ __forceinline__ void store_out(T* out, int d, int h, int c, f32x4 y, float sum) {
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (nothing seen: zeros)
  if (c >= d) return;
  struct {
    T v[4];
  } r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.v[e] = (T)(y[e] * inv);
  __builtin_memcpy(out + (int64_t)h * d + c, &r, sizeof(r));
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

template <typename T, int DP, bool EXACT>
__global__ void __launch_bounds__(64 * paged_waves<DP>(), 1) paged_attention_kernel(const PagedArgs a) {
  constexpr int W = paged_waves<DP>(), UNIT = W * kTile;
  typedef typename Mma<T>::v8 v8;
  constexpr int KS = DP / 32;        // k steps of S^T
  constexpr int DT = DP / 16;        // row tiles of O^T
  constexpr int C = DP / 8;          // 16-byte chunks of a row
  constexpr int VL = C / 2;          // V loads per lane and tile
  constexpr int kRow = 2 * DP + 32;  // LDS bytes of a V row: 16 rows' 32-byte pieces fall on distinct banks
  __shared__ __attribute__((aligned(16))) char v_lds[W][kTile * kRow];
  __shared__ TokenRows rows[W][2][kTile];
  __shared__ float ml[2][W][kHeadTile];
  __shared__ uint32_t ticket;
  static_assert(kTile * kRow >= kHeadTile * DP * 4, "a wave's outputs fit its piece of LDS");

  const int lane0 = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_seq = a.hkv * a.head_tiles;  // (cache head, head tile) pairs of a sequence

  // All units, and this workgroup's run of them.
  const int units0 = span_of<UNIT>(a, lane0 < a.batch ? a.lengths[lane0] : 0).units;
  auto units_of = [&](int b0) __attribute__((always_inline)) {
    const int x = b0 + lane0;
    const int u = b0 == 0 ? units0 : span_of<UNIT>(a, x < a.batch ? a.lengths[x] : 0).units;
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
  Span sp = span_of<UNIT>(a, a.lengths[b]);

  while (at < end) {
    // a segment: units [j0, j1) of one (sequence, cache head, head tile)
    // (opaque per segment: addresses made from it are not kept across segments,
    // nor those of the join across the tiles)
    const int lane = opaque(lane0), lr = lane & 15, lg = lane >> 4;
    const int64_t off = at - seq0;
    const int pair = (int)(off / sp.units);
    const int j0 = (int)(off - (int64_t)pair * sp.units);
    const int j1 = (int)min((int64_t)sp.units, j0 + (end - at));
    const int kvh = pair / a.head_tiles, ht = pair - kvh * a.head_tiles;
    const int head0 = kvh * a.group + ht * kHeadTile;  // first query head
    const int heads = min(kHeadTile, a.group - ht * kHeadTile);
    const int32_t* bt = a.block_table + (int64_t)b * a.table_width;
    const T* kbase = static_cast<const T*>(a.k) + kvh * a.kc_head;
    const T* vbase = static_cast<const T*>(a.v) + kvh * a.vc_head;
    const T* zeros = reinterpret_cast<const T*>(kZeros);

    // Q^T: a lane holds columns 32 s + 8 lg .. + 7 of head lr
    v8 q[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bool in = lr < heads && (EXACT || 32 * s + 8 * lg < a.d);
      const T* p = static_cast<const T*>(a.q) + b * a.q_batch + (head0 + lr) * a.q_head + 32 * s + 8 * lg;
      q[s] = load16<v8>(in ? p : zeros);
    }

    const int tiles = (j1 - j0) * W;
    const int token0 = sp.base + j0 * UNIT;
    auto page_of = [&](int i) __attribute__((always_inline)) {  // of lane's token of tile i; -1: masked
      const int t = token0 + i * kTile + (lane & 31);
      int page = -1;
      if (i < tiles && t >= sp.first && t < sp.len) page = bt[(uint32_t)t / (uint32_t)a.page_size];
      return page;  // (looked at by put_rows, a step later: here it would be waited for)
    };
    auto put_rows = [&](int i, int page) __attribute__((always_inline)) {
      const int t = token0 + i * kTile + (lane & 31);
      const uint32_t slot = (uint32_t)t % (uint32_t)a.page_size;
      TokenRows r{(uint64_t)zeros, (uint64_t)zeros};
      if (page >= 0 && page < a.n_pages)
        r = TokenRows{(uint64_t)(kbase + page * a.kc_page + slot * a.kc_slot), (uint64_t)(vbase + page * a.vc_page + slot * a.vc_slot)};
      if (lane < kTile) rows[wave][(i / W) & 1][lane] = r;
    };
    v8 k[2][KS], v[VL];
    auto load_k = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const T* r = reinterpret_cast<const T*>(rows[wave][(i / W) & 1][16 * h + lr].k) + 8 * lg;
#pragma unroll
        for (int s = 0; s < KS; ++s) k[h][s] = load16<v8>(EXACT || 32 * s + 8 * lg < a.d ? r + 32 * s : zeros);
      }
    };
    // chunk c of a lane: 16-byte piece v_piece(c) of token v_token(c)
    auto v_token = [&](int c) __attribute__((always_inline)) { return 64 % C == 0 ? lane / C + c * (64 / C) : (lane + 64 * c) / C; };
    auto v_piece = [&](int c) __attribute__((always_inline)) { return 64 % C == 0 ? lane % C : (lane + 64 * c) % C; };
    auto load_v = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < VL; ++c) {
        const T* r = reinterpret_cast<const T*>(rows[wave][(i / W) & 1][v_token(c)].v) + 8 * v_piece(c);
        v[c] = load16<v8>(EXACT || 8 * v_piece(c) < a.d ? r : zeros);
      }
    };

    f32x4 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x4{0, 0, 0, 0};
    float m = kLeastScore, l = 0.0f;

    put_rows(wave, page_of(wave));
    wave_lds_fence();
    // (in the loop's order, next pages, keys, values: its waits count loads)
    int page = page_of(wave + W);
    __builtin_amdgcn_sched_barrier(0);
    load_k(wave);
    __builtin_amdgcn_sched_barrier(0);
    load_v(wave);
    __builtin_amdgcn_sched_barrier(0);
    for (int i = wave; i < tiles; i += W) {
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
        for (int c = 0; c < KS; ++c) s[h] = Mma<T>::mul(k[h][c], q[c], s[h]);
      }
      // (sched_barrier: moved up, the loads would take registers of their own)
      __builtin_amdgcn_sched_barrier(0);
      load_k(i + W);

      // lane: head lr, tokens 16 h + 4 lg + e
#pragma unroll
      for (int h = 0; h < 2; ++h) s[h] *= a.scale;
      if (masked) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (masked >> (16 * h + 4 * lg + e) & 1) s[h][e] = -INFINITY;
      }
      float top = m;  // (a NaN is not its maximum, but makes its exponential, so the sums, NaN)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[h][e]);
      top = combine32<MaxOp>(combine16<MaxOp>(top));
      const float keep = __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= keep;
      float x8[8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(s[h][e] - top) * Mma<T>::kUnit;
          l += x;
          x8[4 * h + e] = x;
        }
      v8 p, rest;
#pragma unroll
      for (int e = 0; e < 8; e += 2) Mma<T>::cut(x8[e], x8[e + 1], p, rest, e);
#pragma unroll
      for (int t = 0; t < DT; ++t) o[t] *= keep;

#pragma unroll
      for (int c = 0; c < VL; ++c) {
        *reinterpret_cast<v8*>(v_lds[wave] + v_token(c) * kRow + 16 * v_piece(c)) = v[c];
      }
      wave_lds_fence();
      __builtin_amdgcn_sched_barrier(0);
      load_v(i + W);
      __builtin_amdgcn_sched_barrier(0);
      // V^T: a lane takes column 16 t + lr of tokens 16 h + 4 lg .. + 3
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        i16x4 part[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) i16x4*)(v_lds[wave] + (16 * h + 4 * lg + (lr >> 2)) * kRow + 32 * t +
                                                         8 * (lr & 3)));
        typedef int16_t i16x8 __attribute__((ext_vector_type(8)));
        const i16x8 both = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
        o[t] = Mma<T>::mul(__builtin_bit_cast(v8, both), p, o[t]);
        o[t] = Mma<T>::mul(__builtin_bit_cast(v8, both), rest, o[t]);
        if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (eight reads at a time: registers)
      }
      wave_lds_fence();
    }

    // the waves' states, through LDS
    const int tid = opaque((int)threadIdx.x);
    l = combine32<AddOp>(combine16<AddOp>(l));
    float* ow = reinterpret_cast<float*>(v_lds[wave]);
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(ow + lr * DP + 16 * t + 4 * lg) = o[t];
    if (lane < kHeadTile) ml[0][wave][lane] = m, ml[1][wave][lane] = l;
    __syncthreads();
    T* out = static_cast<T*>(a.out) + ((int64_t)b * a.hq + head0) * a.d;
    if (j0 == 0 && j1 == sp.units) {
      join_waves<DP, W>(tid, heads, W, ml, v_lds[0], kTile * kRow, [&](int h, int c, f32x4 y, float, float sum) {
        store_out(out, a.d, h, c, y, sum);
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
      float* part = a.parts + ((int64_t)blockIdx.x * 2 + (at != start)) * state_floats<DP>();
      join_waves<DP, W>(tid, heads, W, ml, v_lds[0], kTile * kRow, [&](int h, int c, f32x4 y, float top, float sum) {
        put_device(part + 2 * kHeadTile + h * DP + c, y[0], y[1]);
        put_device(part + 2 * kHeadTile + h * DP + c + 2, y[2], y[3]);
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
        const float* parts = a.parts + (g0 * 2 + later) * state_floats<DP>();
        const int64_t next = (2 - later) * state_floats<DP>();  // g0 + 1's, from g0's
        // 64 pieces (a head, 4 columns) of the states are a wave's, or, of few
        // pieces, every PG-th of their states; its loads are in flight together
        const int pieces = heads * (DP / 4), groups = (pieces + 63) / 64, pg = max(1, W / groups);
        auto gather = [&](auto ahead) __attribute__((always_inline)) {
          constexpr int A = decltype(ahead)::value;
          for (int x = wave; x < groups * pg; x += W) {
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
                const float* p = parts + (gz == 0 ? 0 : next + (int64_t)(gz - 1) * 2 * state_floats<DP>());
                pm[z] = get_device(p + 2 * h);
                po[z][0] = get_device(p + 2 * kHeadTile + h * DP + c);
                po[z][1] = get_device(p + 2 * kHeadTile + h * DP + c + 2);
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
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(v_lds[part]) + h * DP + c) = y;
            if (c == 0) ml[0][part][h] = top, ml[1][part][h] = sum;
          }
        };
        if (n <= 4 * pg) gather(std::integral_constant<int, 4>{});
        else gather(std::integral_constant<int, 16>{});
        __syncthreads();
        join_waves<DP, W>(tid, heads, pg, ml, v_lds[0], kTile * kRow, [&](int h, int c, f32x4 y, float, float sum) {
          store_out(out, a.d, h, c, y, sum);
        });
      }
    }
    __syncthreads();
    at += j1 - j0;
    if (at - seq0 == (int64_t)sp.units * per_seq) {
      seq0 = at;
      if (++b < a.batch) sp = span_of<UNIT>(a, a.lengths[b]);
    }
  }
}

// Columns that the kernel's instance for d holds.
inline int padded_d(int64_t d) { return d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

bool paged_sizes_ok(int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  return batch >= 0 && batch <= (1 << 20) && hq >= 1 && hkv >= 1 && hq <= 65536 && hq % hkv == 0 && d >= 8 && d <= 256 && d % 8 == 0;
}

template <typename T, int DP>
void launch_paged(const PagedArgs& a, hipStream_t s) {
  const dim3 grid((uint32_t)device_cu_count());
  if (a.d == DP) hipLaunchKernelGGL((paged_attention_kernel<T, DP, true>), grid, dim3(64 * paged_waves<DP>()), 0, s, a);
  else hipLaunchKernelGGL((paged_attention_kernel<T, DP, false>), grid, dim3(64 * paged_waves<DP>()), 0, s, a);
}

template <typename T>
int dispatch_paged(const PagedArgs& a, hipStream_t s) {
  switch (padded_d(a.d)) {
    case 64: launch_paged<T, 64>(a, s); break;
    case 96: launch_paged<T, 96>(a, s); break;
    case 128: launch_paged<T, 128>(a, s); break;
    case 192: launch_paged<T, 192>(a, s); break;
    default: launch_paged<T, 256>(a, s); break;
  }
  return launch_status();
}

}  // namespace tp

using namespace tp;

extern "C" int64_t tp_paged_attention_workspace_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  if (!paged_sizes_ok(batch, hq, hkv, d)) return -1;
  const int dp = padded_d(d);
  return (int64_t)device_cu_count() * 2 * kHeadTile * (dp + 2) * (int64_t)sizeof(float);
}

extern "C" int64_t tp_paged_attention_counter_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  if (!paged_sizes_ok(batch, hq, hkv, d)) return -1;
  const int64_t tiles = (hq / hkv + kHeadTile - 1) / kHeadTile;
  return batch * hkv * tiles * (int64_t)sizeof(uint32_t);
}

extern "C" int tp_paged_attention(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d, const void* q,
                                  int64_t q_batch, int64_t q_head, const void* k_cache, const int64_t* kc,
                                  const void* v_cache, const int64_t* vc, int64_t n_pages, int64_t page_size,
                                  const int32_t* block_table, int64_t table_width, const int32_t* lengths,
                                  float scale, int64_t window, void* out, void* workspace,
                                  int64_t workspace_bytes, void* counters, int64_t counter_bytes, void* stream) {
  if (dtype != TP_F16 && dtype != TP_BF16) return TP_ERR_BAD_TYPE;
  if (!paged_sizes_ok(batch, hq, hkv, d) || n_pages < 0 || n_pages > 0x7fffffff || page_size < 1 || page_size > (1 << 24) ||
      table_width < 0 || table_width > (1 << 30) || window < 0)
    return TP_ERR_BAD_DIMS;
  if (batch == 0) return TP_OK;
  if (!q || !kc || !vc || !lengths || !out || (n_pages > 0 && (!k_cache || !v_cache)) || (table_width > 0 && !block_table))
    return TP_ERR_NULL_POINTER;  // (empty tensors have no address)
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) return TP_ERR_MISALIGNED;
  if ((q_batch | q_head | kc[0] | kc[1] | kc[2] | vc[0] | vc[1] | vc[2]) & 7) return TP_ERR_MISALIGNED;
  if (((uintptr_t)block_table | (uintptr_t)lengths) & 3) return TP_ERR_MISALIGNED;
  if (!workspace || workspace_bytes < tp_paged_attention_workspace_bytes(batch, hq, hkv, d) || !counters ||
      counter_bytes < tp_paged_attention_counter_bytes(batch, hq, hkv, d))
    return TP_ERR_WORKSPACE;
  if (((uintptr_t)workspace & 15) || ((uintptr_t)counters & 3)) return TP_ERR_MISALIGNED;
  PagedArgs a{};
  a.q = q, a.k = k_cache, a.v = v_cache, a.out = out, a.block_table = block_table, a.lengths = lengths;
  a.parts = static_cast<float*>(workspace), a.counters = static_cast<uint32_t*>(counters);
  a.q_batch = q_batch, a.q_head = q_head;
  a.kc_page = kc[0], a.kc_slot = kc[1], a.kc_head = kc[2], a.vc_page = vc[0], a.vc_slot = vc[1], a.vc_head = vc[2];
  a.n_pages = n_pages, a.table_width = table_width, a.window = window;
  a.batch = (int)batch, a.hq = (int)hq, a.hkv = (int)hkv, a.group = (int)(hq / hkv), a.d = (int)d;
  a.head_tiles = (a.group + kHeadTile - 1) / kHeadTile;
  a.page_size = (int)page_size, a.scale = scale * 1.44269504088896340736f;
  hipStream_t s = (hipStream_t)stream;
  return dtype == TP_F16 ? dispatch_paged<f16_t>(a, s) : dispatch_paged<bf16_t>(a, s);
}
