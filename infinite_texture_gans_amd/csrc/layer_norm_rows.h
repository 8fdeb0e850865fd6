// Included by layer_norm.hip; compiles for the host too.
#pragma once
#include <type_traits>
#include "itg_common.h"

namespace {

// Rows of a layer norm held in registers: which values a thread holds, and how it reads them.  A row of c values is cut into vectors
// of V (16 bytes; single values where c < V); TPR threads share a row and a thread holds the R vectors tid, tid + TPR, ...  The last
// vector of a row that V does not divide either starts at c - V and masks what it shares with its neighbour (both write the same
// values there), or, in rows with zero padding behind the channels, lies where it belongs and masks the padding: gamma and beta
// have no such padding, and that vector of theirs is read up to its last value.  Vector loads and stores need the element's alignment only.
struct LnV { int nv, off_last, lo_last, hi_last; };      // vectors per row; start of the last one and its valid elements [lo, hi)

__host__ __device__ inline LnV ln_vectors(int c, int pad, int V) {
  LnV v;
  v.nv = (c + V - 1) / V;
  const bool padded = pad > 0 && pad < V && (c + pad) % V == 0;
  v.off_last = padded ? (v.nv - 1) * V : c - V;
  v.lo_last = (v.nv - 1) * V - v.off_last;
  v.hi_last = padded ? c - v.off_last : V;
  return v;
}

// vector i of a row: where it starts, and its valid elements [lo, hi); none (hi = 0) behind the row's last one, whose place it gets
__host__ __device__ inline void ln_place(const LnV& v, int i, int V, int& off, int& lo, int& hi) {
  off = i < v.nv - 1 ? i * V : v.off_last;
  lo = i < v.nv - 1 ? 0 : v.lo_last;
  hi = i < v.nv - 1 ? V : i < v.nv ? v.hi_last : 0;
}

template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };

// V values as they lie in memory, in 32-bit words (a Pack of 16-bit values takes a register each)
template <typename T, int V> struct Held {
  static constexpr int N = (V * (int)sizeof(T) + 3) / 4;
  uint32_t w[N];
  __device__ __forceinline__ float at(int e) const {
    if (sizeof(T) == 4) return __builtin_bit_cast(float, w[e]);
    return (float)__builtin_bit_cast(T, (typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type)(w[e / 2] >> (16 * (e & 1))));
  }
  __host__ __device__ __forceinline__ void load(const T* q) {
    struct __attribute__((packed, aligned(sizeof(T)))) Words { uint32_t w[N]; };
    if (V * sizeof(T) % 4 == 0) {
      const Words u = *reinterpret_cast<const Words*>(q);
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = u.w[i];
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(q);
    }
  }
  // The first `hi` >= 1 of the V values from `q` on and zeros behind them, of an array that has V values up to there: read as the V
  // values in front of q + hi and moved down, without a branch (value by value it takes up to 57 registers more, which are spills)
  __host__ __device__ __forceinline__ void load_first(const T* q, int hi) {
    const int down = V - hi;
    load(q - down);
#pragma unroll
    for (int step = 1; step < V; step *= 2) {
      constexpr int PER = 4 / (int)sizeof(T);                // values of a word
      const bool moves = (down & step) != 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t next = i + 1 < N ? w[i + 1] : 0u;
        const uint32_t from = step < PER ? w[i] >> 16 | next << 16 : i + step / PER < N ? w[i + step / PER] : 0u;
        w[i] = moves ? from : w[i];
      }
    }
  }
  // the compiler takes the values for changed: what is computed from them again is not carried over in registers instead
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int i = 0; i < N; ++i) asm("" : "+v"(w[i]));
  }
};

}  // namespace
