// Log probabilities of given tokens, entropies and the most likely tokens of
// rows of logits.  With m the largest logit of a row and
//
//   s = sum e^(x - m) - 1,  a = sum (x - m) e^(x - m)
//
// (the largest itself is the 1), log p(x) = x - m - log(1 + s) and the entropy is
// log(1 + s) - a / (1 + s), both terms at least 0: nothing cancels, and a row that
// is nearly certain keeps the relative accuracy of what it is from being so.
//
// A wave takes a segment of a row, 2048 logits at a time in registers; each lane
// keeps sums of its own, scaled by a power of two near its own largest.  The last
// wave of a row to finish joins the segments'.  The one lane that holds the row's
// largest would lose what is small beside it: its logits (one in 64 of its
// segment) are read again and summed without the largest.
//
// The most likely tokens: a wave leaves the largest of every 128 logits too.  The
// k-th largest of 128 groups' largest of those is a bound that the k likeliest
// reach; the few sets of 128 that reach it are read again, and the logits that
// reach it are ranked by (value, lower token first) as one whole number.
//
// Logits are read once, some 9 vector instructions for each (its type, exponential, two
// sums, largest): bound by HBM and by issue alike (2047 x 151936 bf16: 119 us = 5.2 TB/s, with
// the 20 likeliest 159; 4 rows with 5 17 us, a chain of loads, join, sets and ranking).
#include "tp_ops_common.h"

namespace tp {

constexpr int kSet = 128;          // logits whose largest is kept
constexpr int kVectors = 4;        // of 8 logits that a lane holds
constexpr int kPiece = 512 * kVectors;
constexpr int kPieceSets = kPiece / kSet;
constexpr int kState = 8;          // floats of a segment's state (7 of use)
constexpr int kSegments = 128;     // of a row, at most: two states a lane
constexpr int kSetRows = 20;       // of 64 sets in registers (rows of up to 163840 logits: all)
constexpr int kIdBits = 24;        // of a token in an order key
constexpr int kHeld = 256;         // candidates of a row held at once
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
// Powers of two that sums are about, at most and at least.  An exponent fma(x, log2e,
// -power) is exact to a rounding of its own size, but the power itself is a rounded
// product: within 1 of a lane's largest up to 2^24, past that by as much as the
// product's last bits, and the largest's exponential could overflow (of -1e10 it would
// be 2^439).  About -kMostPower logits far below it count as 0, as they do beside a
// row's largest above -kHuge: kMostPower - kHuge log2e = 2.3e6 powers of two.
// (Rows whose largest is kHuge and above are rare: 64 x 151936 of -1e9 alone, fp32, with
// 5 likeliest 430 us, of which the ranking of so many equals is 280.)
constexpr float kMostPower = 8388608.0f;
constexpr float kHuge = 4194304.0f;  // largest logits of this size and above: a way of their own

// The order of values: NaN above everything, negative zero with zero.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  const uint32_t o = u >> 31 ? ~u : u | 0x80000000u;
  return x != x ? 0xffffffffu : o;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __builtin_bit_cast(float, order >> 31 ? order & 0x7fffffffu : ~order);
}
// Larger logits first, of equal ones the lower token.
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  return (uint64_t)order_of(x) << kIdBits | (uint32_t)((1 << kIdBits) - 1 - token);
}

struct LogprobArgs {
  const void* logits;
  const int64_t* tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  float* states;       // [rows][segments][kState]
  float* sets;         // [rows][pieces * kPieceSets]: their largest
  uint32_t* counters;  // per row: segments done; zero between launches
  int64_t rows, ld;
  int vocab, top, pieces, span, segments;  // span: pieces of a segment
};

__device__ __forceinline__ void put_agent(float* p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get_agent(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// (of loaded values the compiler would first quiet each: an instruction more)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

struct PlainMaxOp {
  __device__ __forceinline__ static float of(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
  }
};

// Eight logits as loaded, from a 16-byte aligned address; those whose place is
// outside [from, to) are -infinity.
template <typename T>
struct Eight {
  u32x4 w[sizeof(T) / 2];
  // (pieces of 16 bytes; in place of those from place `to` on the last before it,
  // without a branch, so that several loads are in flight)
  __device__ __forceinline__ void load(const T* p, int place, int to) {
    constexpr int each = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / each; ++i) w[i] = *reinterpret_cast<const u32x4*>(p + min(place + each * i, (to - 1) & ~(each - 1)));
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t x = w[e / 4][e % 4];  // (a bit_cast of the element itself reads element 0)
      return __builtin_bit_cast(float, x);
    } else if constexpr (__is_same(T, bf16_t)) {
      const uint32_t x = w[0][e / 2];
      return __builtin_bit_cast(float, e % 2 ? x & 0xffff0000u : x << 16);
    } else {
      return (float)__builtin_bit_cast(f16_t, (uint16_t)(w[0][e / 2] >> (e % 2 * 16)));
    }
  }
  __device__ __forceinline__ float most() const {  // (of numbers)
    return max3(max3(get(0), get(1), get(2)), max3(get(3), get(4), get(5)), max3(get(6), get(7), get(7)));
  }
  // element e + 1 becomes element e
  __device__ __forceinline__ void shift() {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 7; ++e) w[e / 4][e % 4] = w[(e + 1) / 4][(e + 1) % 4];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[0][i] = __builtin_amdgcn_alignbyte(i < 3 ? w[0][i < 3 ? i + 1 : 3] : 0, w[0][i], 2);
    }
  }
  __device__ __forceinline__ void hide(int e) {
    if constexpr (sizeof(T) == 4) {
      w[e / 4][e % 4] = 0xff800000u;
    } else {
      const uint32_t inf = __is_same(T, bf16_t) ? 0xff80u : 0xfc00u, x = w[0][e / 2];
      w[0][e / 2] = e % 2 ? (x & 0xffffu) | inf << 16 : (x & 0xffff0000u) | inf;
    }
  }
  __device__ __forceinline__ void keep(int place, int from, int to) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (place + e < from || place + e >= to) hide(e);
  }
};

// A row: logit i is at place i + shift of 16-byte aligned memory.
template <typename T>
struct Row {
  const T* base;
  int shift, end;  // places [shift, end)
  __device__ __forceinline__ Row(const LogprobArgs& a, int64_t row) {
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    shift = (int)((uintptr_t)x / sizeof(T)) & (int)(16 / sizeof(T) - 1);
    base = x - shift;
    end = a.vocab + shift;
  }
  // 8 places from a multiple of 8 on, those outside the row -infinity
  __device__ __forceinline__ Eight<T> load(int place) const {
    Eight<T> v;
    v.load(base, place, end);
    v.keep(place, shift, end);
    return v;
  }
};

// The largest t with at least k of the wave's keys at t or above (fewer than k
// keys: 0; keys are above 0).  Only the bits in which keys differ are looked for.
template <typename K, int N>
__device__ __forceinline__ K kth_key(const K (&keys)[N], int k) {
  int count = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) count += __builtin_popcountll(__ballot(keys[i] > 0));
  if (count < k) return 0;
  K all = 0, both = ~(K)0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    all |= keys[i];
    both &= keys[i] > 0 ? keys[i] : ~(K)0;
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    all |= (K)__shfl_xor(all, o);
    both &= (K)__shfl_xor(both, o);
  }
  K t = both;
  for (K left = all & ~both; left;) {
    const K bit = (K)1 << (8 * sizeof(K) - 1 - (sizeof(K) == 8 ? __builtin_clzll(left) : __builtin_clz((uint32_t)left)));
    left &= ~bit;
    const K next = t | bit;  // (bits below are those that all keys have: no key between is passed over)
    count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __builtin_popcountll(__ballot(keys[i] >= (next & ~(bit - 1))));
    if (count >= k) t = next;
  }
  return t;
}

// Appends the keys of the lanes that take, after the n held.
__device__ __forceinline__ int append(uint64_t* held, int n, uint64_t key, bool take) {
  const uint64_t all = __ballot(take);
  if (take) held[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0))] = key;
  return n + __builtin_popcountll(all);
}

// The k largest of n (up to kHeld) held keys, moved to the front; the least of them.
__device__ __forceinline__ uint64_t keep_largest(uint64_t* held, int n, int k, int lane) {
  constexpr int N = kHeld / 64;
  uint64_t keys[N];
  wave_lds_fence();
#pragma unroll
  for (int i = 0; i < N; ++i) keys[i] = lane + 64 * i < n ? held[lane + 64 * i] : 0;
  const uint64_t t = kth_key(keys, k);
  wave_lds_fence();
  int at = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) at = append(held, at, keys[i], keys[i] >= t && keys[i] > 0);
  wave_lds_fence();
  return t;
}

// The row's most likely tokens, by one wave.  log_sum: what log probabilities are
// less than logit - largest by; odd: the row holds NaN or +infinity.
template <typename T>
__device__ __forceinline__ void rank_row(const LogprobArgs& a, int64_t row, const Row<T>& x, uint64_t* held, uint16_t* list,
                                         int lane, float largest, float log_sum, bool none, bool odd) {
  const int sets = (x.end + kSet - 1) / kSet;
  const float* tops = a.sets + row * a.pieces * kPieceSets;
  float tops_at[kSetRows];
  auto load_sets = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kSetRows; ++i) tops_at[i] = get_agent(tops + min(s0 + 64 * i + lane, sets - 1));
  };
  // a bound: the largest of the sets of a lane, of even and of odd rows
  uint64_t least = 0;
  if (!odd) {
    uint32_t best[2] = {0, 0};
    for (int s0 = 0; s0 < sets; s0 += 64 * kSetRows) {
      load_sets(s0);
#pragma unroll
      for (int i = 0; i < kSetRows; ++i)
        if (s0 + 64 * i + lane < sets) best[i & 1] = max(best[i & 1], order_of(tops_at[i]));
    }
    least = (uint64_t)kth_key(best, a.top) << kIdBits;
  }
  int n = 0;
  for (int s0 = 0; s0 < sets; s0 += 64 * kSetRows) {
    // the sets that may reach it, listed
    if (sets > 64 * kSetRows || odd) load_sets(s0);
    int listed = 0;
#pragma unroll
    for (int i = 0; i < kSetRows; ++i) {
      const int set = s0 + 64 * i + lane;
      const bool in = set < sets && (odd || key_of(tops_at[i], max(set * kSet - x.shift, 0)) >= least);
      const uint64_t all = __ballot(in);
      if (in) list[listed + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0))] = set - s0;
      listed += __builtin_popcountll(all);
    }
    wave_lds_fence();
    // their logits that do: 16 lanes a set, 16 sets in flight
    for (int l = 0; l < listed; l += 16) {
      int place[4];
      Eight<T> v[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = l + 4 * g + (lane >> 4);
        place[g] = at < listed ? (s0 + list[at]) * kSet + 8 * (lane & 15) : x.end;
        v[g].load(x.base, place[g], x.end);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g)
        for (int e = 0; e < 8; ++e, v[g].shift()) {
          const uint64_t key = key_of(v[g].get(0), place[g] + e - x.shift);
          const bool take = place[g] + e >= x.shift && place[g] + e < x.end && key >= least;
          if (__any(take)) {
            if (n > kHeld - 64) {
              least = keep_largest(held, n, a.top, lane);
              n = a.top;
            }
            n = append(held, n, key, take && key >= least);
          }
        }
    }
    wave_lds_fence();
  }
  if (n > 64) {
    keep_largest(held, n, a.top, lane);
    n = a.top;
  }
  const uint64_t key = lane < n ? held[lane] : 0;
  int rank = 0;
  for (int i = 0; i < n; ++i) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)key, i), hi = __builtin_amdgcn_readlane((uint32_t)(key >> 32), i);
    rank += ((uint64_t)hi << 32 | lo) > key;
  }
  if (lane < n && rank < a.top) {
    const float y = value_of((uint32_t)(key >> kIdBits));
    a.top_tokens[row * a.top + rank] = (1 << kIdBits) - 1 - (int)(key & ((1 << kIdBits) - 1));
    a.top_logprobs[row * a.top + rank] = odd ? __builtin_nanf("") : none ? -INFINITY : y - largest - log_sum;
  }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(256) token_logprobs_kernel(const LogprobArgs a) {
  __shared__ uint64_t held[TOP ? 4 : 1][TOP ? kHeld : 1];
  __shared__ uint16_t list[TOP ? 4 : 1][TOP ? 64 * kSetRows : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t at = blockIdx.x * 4 + wave;
  const uint32_t r32 = at / (uint32_t)a.segments;
  const int segment = (int)(at - r32 * (uint32_t)a.segments);
  const int64_t row = r32;
  if (row >= a.rows) return;
  const Row<T> x(a, row);

  // The segment.  sum = sum 2^(x log2e - power) and off = sum of those times their
  // exponents, about the lane's own power (a whole number, so that a larger one
  // scales both exactly); sum is NaN where the lane meets NaN, and may be +infinity
  // where the row's largest is kHuge and above.
  float largest = -INFINITY, power = -kMostPower, sum = 0.0f, off = 0.0f;
  const int first = segment * a.span, last = min(first + a.span, a.pieces);
  for (int piece = first; piece < last; ++piece) {
    const int place0 = piece * kPiece + 8 * lane;
    Eight<T> v[kVectors];
#pragma unroll
    for (int j = 0; j < kVectors; ++j) v[j].load(x.base, place0 + 512 * j, x.end);
    if ((piece == 0 && x.shift > 0) || (piece + 1) * kPiece > x.end) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j) v[j].keep(place0 + 512 * j, x.shift, x.end);
    }
    float of_set = 0.0f;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      float m = v[j].most();
      largest = PlainMaxOp::of(largest, m);
      if constexpr (TOP) {
        m = reduce16<PlainMaxOp>(m);
        if ((lane & 15) == j) of_set = m;
      }
    }
    if constexpr (TOP) {
      if ((lane & 15) < kVectors)
        put_agent(a.sets + (row * a.pieces + piece) * kPieceSets + (lane & 15) * 4 + (lane >> 4), of_set);
    }
    const float up = fminf(fmaxf(ceilf(largest * kLog2e), -kMostPower), kMostPower), scale = __builtin_amdgcn_exp2f(power - up);
    off = scale * __builtin_fmaf(power - up, sum, off);
    sum *= scale;
    power = up;
    float s = 0.0f, o = 0.0f;
#pragma unroll
    for (int j = 0; j < kVectors; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __builtin_fmaf(v[j].get(e), kLog2e, -up), p = __builtin_amdgcn_exp2f(y);
        s += p;
        o = __builtin_fmaf(y, p, o);
      }
    if (__any(o != o && s == s)) {  // (-infinity times its weight of 0)
      o = 0.0f;
      float again = up;
      asm volatile("" : "+v"(again));  // (else these are computed beside the others, in case)
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = __builtin_fmaf(v[j].get(e), kLog2e, -again);
          o = __builtin_fmaf(fmaxf(y, -200.0f), __builtin_amdgcn_exp2f(y), o);
        }
    }
    sum += s;
    off += o;
  }

  // the wave's, and without the lane that holds its largest
  float* state = a.states + (row * a.segments + segment) * kState;
  {
    const float most = reduce64<MaxOp>(largest), all = reduce64<MaxOp>(power), f = __builtin_amdgcn_exp2f(power - all);
    const uint64_t is = __ballot(largest == most);
    const int holder = is ? __builtin_ctzll(is) : 0;
    off = f * __builtin_fmaf(power - all, sum, off);
    sum *= f;
    const float others = reduce64<AddOp>(lane == holder ? 0.0f : sum), others_off = reduce64<AddOp>(lane == holder ? 0.0f : off);
    sum = reduce64<AddOp>(sum);
    off = reduce64<AddOp>(off);
    if (lane < 7) {
      const float mine = lane == 0 ? most : lane == 1 ? all : lane == 2 ? sum : lane == 3 ? off : lane == 4 ? others
                       : lane == 5 ? others_off : (float)holder;
      put_agent(state + lane, mine);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (a.segments > 1) {
    uint32_t done = 0;
    if (lane == 0) done = __hip_atomic_fetch_add(a.counters + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    done = __builtin_amdgcn_readfirstlane(done);
    asm volatile("" ::: "memory");
    if (done != (uint32_t)a.segments - 1) return;
    if (lane == 0) __hip_atomic_store(a.counters + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }

  // The row's: all segments' sums about the largest of all.
  const float* states = a.states + row * a.segments * kState;
  float st[2][7];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int c = 0; c < 7; ++c) st[i][c] = get_agent(states + min(lane + 64 * i, a.segments - 1) * kState + c);
  if (lane >= a.segments) st[0][0] = -INFINITY, st[0][2] = 0.0f;
  if (lane + 64 >= a.segments) st[1][0] = -INFINITY, st[1][2] = 0.0f;
  const float top = reduce64<MaxOp>(fmaxf(st[0][0], st[1][0]));
  const bool none = top == -INFINITY;
  const bool odd = __any(st[0][2] != st[0][2] || st[1][2] != st[1][2]) || top == INFINITY;
  float rest = 0.0f, diff = 0.0f, count = 0.0f;
  if (odd || none) {
  } else if (fabsf(top) < kHuge) {
    // the first segment, then its first lane, that holds the largest
    const uint64_t low = __ballot(st[0][0] == top), high = __ballot(st[1][0] == top);
    const int holder = low ? __builtin_ctzll(low) : 64 + __builtin_ctzll(high);
    const float its_lane = low ? __shfl(st[0][6], holder) : __shfl(st[1][6], holder - 64);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float y = -__builtin_fmaf(top, kLog2e, -st[i][1]), f = __builtin_amdgcn_exp2f(y);
      if (lane + 64 * i < a.segments && f > 0.0f) {
        const bool is = lane + 64 * i == holder;
        const float si = is ? st[i][4] : st[i][2], oi = is ? st[i][5] : st[i][3];
        diff += f * __builtin_fmaf(y, si, oi);
        rest += f * si;
      }
    }
    // its logits again: vector i of the segment's at 512 i
    const int begin = holder * a.span * kPiece + 8 * (int)its_lane, vectors = (min((holder + 1) * a.span, a.pieces) - holder * a.span) * kVectors;
    for (int i = lane; i < vectors; i += 64) {
      Eight<T> u;
      u.load(x.base, begin + 512 * i, x.end);
      u.keep(begin + 512 * i, x.shift, x.end);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = u.get(e), y = (f - top) * kLog2e, p = __builtin_amdgcn_exp2f(y);
        count += f == top ? 1.0f : 0.0f;
        rest += f == top ? 0.0f : p;
        diff = __builtin_fmaf(fmaxf(y, -200.0f), p, diff);
      }
    }
  } else {
    // (their power is no whole number near them: the whole row about its largest)
    for (int place = 8 * lane; place < x.end; place += 512) {
      Eight<T> u;
      u.load(x.base, place, x.end);
      u.keep(place, x.shift, x.end);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = u.get(e), y = (f - top) * kLog2e, p = __builtin_amdgcn_exp2f(y);
        count += f == top ? 1.0f : 0.0f;
        rest += f == top ? 0.0f : p;
        diff = __builtin_fmaf(fmaxf(y, -200.0f), p, diff);
      }
    }
  }
  const float others = reduce64<AddOp>(rest) + (reduce64<AddOp>(count) - 1.0f);
  diff = reduce64<AddOp>(diff) * kLn2;
  const float log_sum = log1pf(others);
  if (lane == 0) {
    const float nan = __builtin_nanf("");
    a.entropy[row] = odd ? nan : none ? 0.0f : log_sum - diff / (1.0f + others);
    if (a.tokens) {
      const int64_t t = a.tokens[row];
      float y = 0.0f;
      if (t >= 0) {
        y = nan;
        if (t < a.vocab && !odd) y = none ? -INFINITY : (float)x.base[t + x.shift] - top - log_sum;
      }
      a.logprobs[row] = y;
    }
  }
  if constexpr (TOP) rank_row<T>(a, row, x, held[wave], list[wave], lane, top, log_sum, none, odd);
}

// (room for the up to 7 places before a row's first logit)
inline int64_t logprob_pieces(int64_t vocab) { return (vocab + 7 + kPiece - 1) / kPiece; }
// Pieces of a segment: so few that kWaves waves and more have work, no fewer: a wave's
// start, its sums' joins and the row's ticket cost as much as several pieces (151936
// columns, 5 likeliest, 1024 / 2048 / 4096 / 8192 / 16384 waves: 4 rows 17 us all, 100 25 /
// 26 / 34 / 59, 256 31 / 30 / 34 / 43 / 53, 600 62 / 51 / 54 / 56; 2047 rows, 20 likeliest
// 160 / 159 / 168 / 173 / 180).
constexpr int64_t kWaves = 2048;
inline int64_t logprob_span(int64_t rows, int64_t vocab) {
  const int64_t pieces = logprob_pieces(vocab), want = (kWaves + rows - 1) / rows, most = want < kSegments ? want : kSegments;
  return (pieces + most - 1) / most;
}
inline int64_t logprob_segments(int64_t rows, int64_t vocab) {
  const int64_t span = logprob_span(rows, vocab);
  return (logprob_pieces(vocab) + span - 1) / span;
}

template <typename T>
int launch_logprobs(const LogprobArgs& a, hipStream_t s) {
  const dim3 grid((uint32_t)((a.rows * a.segments + 3) / 4)), block(256);
  if (a.top) hipLaunchKernelGGL((token_logprobs_kernel<T, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((token_logprobs_kernel<T, false>), grid, block, 0, s, a);
  return launch_status();
}

inline bool logprob_sizes_ok(int64_t rows, int64_t vocab, int64_t top) {
  return rows >= 0 && rows <= (1 << 24) && vocab >= 1 && vocab <= (1 << kIdBits) - 8 && top >= 0 && top <= 64 && top <= vocab;
}

}  // namespace tp

using namespace tp;

extern "C" int64_t tp_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top) {
  if (!logprob_sizes_ok(rows, vocab, top)) return -1;
  if (rows == 0) return 0;
  return 4 * rows * (kState * logprob_segments(rows, vocab) + (top ? kPieceSets * logprob_pieces(vocab) : 0));
}

extern "C" int64_t tp_token_logprobs_counter_bytes(int64_t rows, int64_t vocab, int top) {
  return logprob_sizes_ok(rows, vocab, top) ? rows * (int64_t)sizeof(uint32_t) : -1;
}

extern "C" int tp_token_logprobs(int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                                 const int64_t* tokens, float* logprobs, float* entropy, int top, float* top_logprobs,
                                 int64_t* top_tokens, void* workspace, int64_t workspace_bytes, void* counters,
                                 int64_t counter_bytes, void* stream) {
  if (!dtype_ok(dtype)) return TP_ERR_BAD_TYPE;
  if (!logprob_sizes_ok(rows, vocab, top) || ld < 0) return TP_ERR_BAD_DIMS;
  if (rows == 0) return TP_OK;
  if (!logits || !entropy || (tokens && !logprobs) || (top && (!top_logprobs || !top_tokens))) return TP_ERR_NULL_POINTER;
  if (((uintptr_t)logits & (dtype_bytes(dtype) - 1)) || (((uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)top_logprobs) & 3) ||
      (((uintptr_t)tokens | (uintptr_t)top_tokens) & 7))
    return TP_ERR_MISALIGNED;
  if (!workspace || workspace_bytes < tp_token_logprobs_workspace_bytes(rows, vocab, top) || !counters ||
      counter_bytes < tp_token_logprobs_counter_bytes(rows, vocab, top))
    return TP_ERR_WORKSPACE;
  if (((uintptr_t)workspace & 15) || ((uintptr_t)counters & 3)) return TP_ERR_MISALIGNED;
  LogprobArgs a{};
  a.logits = logits, a.tokens = tokens, a.logprobs = logprobs, a.entropy = entropy;
  a.top_logprobs = top_logprobs, a.top_tokens = top_tokens, a.rows = rows, a.ld = ld, a.vocab = (int)vocab, a.top = top;
  a.pieces = (int)logprob_pieces(vocab), a.span = (int)logprob_span(rows, vocab), a.segments = (int)logprob_segments(rows, vocab);
  a.states = static_cast<float*>(workspace), a.sets = a.states + rows * a.segments * kState;
  a.counters = static_cast<uint32_t*>(counters);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TP_F16) return launch_logprobs<f16_t>(a, s);
  if (dtype == TP_BF16) return launch_logprobs<bf16_t>(a, s);
  return launch_logprobs<float>(a, s);
}
