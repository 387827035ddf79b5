// What the decoder operators (norm, rotary positions, 8-bit product, paged
// attention) share: element types, unaligned vectors, reductions across lanes.
#pragma once

#include "tp_common.h"

namespace tp {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Casts between element types and fp32; f32 -> f16 / bf16 round to nearest even.
template <typename T>
struct Vec {
  T v[8];
};

// 8 elements at any element-aligned address (gfx950 takes global accesses of
// any byte alignment; the compiler makes one 16-byte access of a 2-byte type).
template <typename T>
__device__ __forceinline__ Vec<T> load8(const T* p) {
  Vec<T> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const Vec<T>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}

// The same past the caches: of what is read once and is too large to be in them,
// and of what is written once.
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x4 u32x4_words __attribute__((aligned(4)));
template <typename T>
__device__ __forceinline__ Vec<T> load8_once(const T* p) {
  u32x4 w[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p) + i);
  Vec<T> r;
  __builtin_memcpy(&r, w, sizeof(r));
  return r;
}
template <typename T>
__device__ __forceinline__ void store8_once(T* p, const Vec<T>& r) {
  u32x4 w[sizeof(T) / 2];
  __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4_any*>(p) + i);
}

// 4 N bytes at any alignment: the words that hold them, loaded as they lie (a
// word that holds a byte of a row is memory), and moved over by the address's
// last bits.  Loads off their words take several times as long: the product of
// 16 rows and 2560 x 9727 e4m3 weights 40 us against 15, the norm of 8191 x 9727
// fp16 79 against 72 (stores off their words cost little).  ONCE: past the caches.
template <int N>
struct Unaligned {
  static_assert(N % 4 == 0, "");
  u32x4 at[N / 4];
  uint32_t next;

  // (own: with the word behind; else the caller gets it from who has it)
  template <bool ONCE = false>
  __device__ __forceinline__ void load(const void* p, bool own = true) {
    const uint32_t s = (uint32_t)(uintptr_t)p & 3;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const char*>(p) - s);
#pragma unroll
    for (int x = 0; x < N / 4; ++x) {
      const u32x4_words* w = reinterpret_cast<const u32x4_words*>(q) + x;
      at[x] = ONCE ? __builtin_nontemporal_load(w) : *w;
    }
    next = 0;
    if (own) next = q[s ? N : N - 1];  // (at s = 0 not used)
  }
  // The first `left` bytes, then zeros.
  __device__ __forceinline__ void load_first(const void* p, int left) {
    const uint32_t s = (uint32_t)(uintptr_t)p & 3;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const char*>(p) - s);
    const int n = left > 0 ? left + (int)s : 0;
#pragma unroll
    for (int x = 0; x < N; ++x) at[x / 4][x % 4] = 4 * x < n ? q[x] : 0;
    next = 4 * N < n ? q[N] : 0;
#pragma unroll
    for (int x = 0; x <= N; ++x) {
      const int in = n - 4 * x;  // bytes of the row in this word
      const uint32_t keep = in >= 4 ? ~0u : in <= 0 ? 0u : (1u << (8 * in)) - 1;
      if (x < N) at[x / 4][x % 4] &= keep;
      else next &= keep;
    }
  }
  // Word x of what was loaded; s: the address's last two bits.
  __device__ __forceinline__ uint32_t word(int x, uint32_t s) const {
    return __builtin_amdgcn_alignbyte(x + 1 < N ? at[(x + 1) / 4][(x + 1) % 4] : next, at[x / 4][x % 4], s);
  }
};

// A launch holds less than 2^32 threads.
inline bool grid_fits(int64_t blocks, int threads) { return blocks * threads <= 0xffffffffll; }

// Lane i takes lane i + 1's value (wave_shl:1), lane 63 keeps its own.
__device__ __forceinline__ uint32_t from_next_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x130, 0xF, 0xF, false);
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}

struct AddOp {
  __device__ __forceinline__ static float of(float a, float b) { return a + b; }
};
struct MaxOp {
  __device__ __forceinline__ static float of(float a, float b) { return fmaxf(a, b); }
};
// The larger of two; NaN where either is (v_max_f32 drops a NaN).
struct MaxNanOp {
  __device__ __forceinline__ static float of(float a, float b) { return a > b || a != a ? a : b; }
};

// Over the 16 lanes of a row, in every lane: lane xor 1, xor 2, then (the
// values being equal within groups) the half-row and the row mirror.
template <typename Op>
__device__ __forceinline__ float reduce16(float v) {
  v = Op::of(v, dpp<0xB1>(v));
  v = Op::of(v, dpp<0x4E>(v));
  v = Op::of(v, dpp<0x141>(v));
  return Op::of(v, dpp<0x140>(v));
}

// The value of the lane 16 (or 32) away, combined: both results of a permlane
// swap of v with itself hold one of the two rows (halves) in every lane.
template <typename Op>
__device__ __forceinline__ float combine16(float v) {
  const uint32_t x = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return Op::of(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
template <typename Op>
__device__ __forceinline__ float combine32(float v) {
  const uint32_t x = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return Op::of(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Over the 64 lanes of a wave, in every lane.
template <typename Op>
__device__ __forceinline__ float reduce64(float v) {
  return combine32<Op>(combine16<Op>(reduce16<Op>(v)));
}

inline bool dtype_ok(int dtype) { return dtype == TP_F16 || dtype == TP_BF16 || dtype == TP_F32; }
inline int dtype_bytes(int dtype) { return dtype == TP_F32 ? 4 : 2; }

}  // namespace tp
