// Included by layer_norm.hip; compiles for the host too.
#pragma once
#include <type_traits>
#include "itg_common.h"

namespace {

// the padding behind a row completes its last vector
__host__ __device__ inline bool ln_padded(int c, int pad, int V) { return pad > 0 && pad < V && (c + pad) % V == 0; }

// Rows of a layer norm held in registers: which values a thread holds, and how it reads them.  A row of c values is cut into vectors
// of V (16 bytes; single values where c < V); TPR threads share a row and a thread holds the R vectors tid, tid + TPR, ...  The last
// vector of a row that V does not divide either starts at c - V and masks what it shares with its neighbour (both write the same
// values there), or, in rows with zero padding behind the channels, lies where it belongs and masks the padding: gamma and beta
// have no such padding, and that vector of theirs is read up to its last value.  Vector loads and stores need the element's alignment only.
struct LnV { int nv, off_last, lo_last, hi_last; };      // vectors per row; start of the last one and its valid elements [lo, hi)

__host__ __device__ inline LnV ln_vectors(int c, int pad, int V) {
  LnV v;
  v.nv = (c + V - 1) / V;
  const bool padded = ln_padded(c, pad, V);
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

// ---- the backward pass's kernel for a call, and the shares of dw | db that it leaves
constexpr int LN_CHUNKS = 1024;      // at most this many from rows in registers

// Threads per row, 0: the kernels for any length.  Up to two vectors in a wave (65536 x 1023 bf16 96 us, in two waves of one each
// 120, where 1024 shares of dw | db are 8 waves a CU), then one of 8 or two of 4, as a thread keeps six values per channel it holds;
// at two of 8 its row stays in 16 bits, see there.
// A row in registers is read once, but every workgroup leaves a share of dw | db, 16 bytes a channel written and read, where the
// kernels for any length read the row three times and leave a share per 8 rows: those for few long rows (bf16, 8192 channels:
// 256 rows 24.4 us in registers, 16.0 swept; 768 rows 25.5, 30.5; 16384 channels: 512 rows 43, 33; 1536 rows 59, 81)
inline int ln_bwd_threads(int64_t rows, int c, int pad, int V) {
  const int nv = (c + V - 1) / V, K = V == 8 ? 1 : 2;      // K: vectors per thread of the workgroup sizes
  const bool few = c >= 8192 && rows * 16 < c;
  if (c < V && !ln_padded(c, pad, V)) return c <= 4 ? 4 : 8;
  for (int t = 4; t <= 64; t *= 2)
    if (nv <= t) return t;
  if (nv <= 128) return 64;
  for (int t = 128 * (3 - K); t <= 512; t *= 2)
    if (nv <= t * K) return t;
  return nv <= 2048 && !few ? 1024 : 0;
}

// rows in registers: every CU has a workgroup before one gets fewer than four turns: a share costs a write and a read of 2 c floats
inline int ln_bwd_groups(int64_t rows, int threads) {
  const int nt = threads > 64 ? threads : 256, most = 256 * (1024 / nt) < LN_CHUNKS ? 256 * (1024 / nt) : LN_CHUNKS;
  const int64_t need = (rows + nt / threads - 1) / (nt / threads), few = need / 4 > 256 ? need / 4 : 256, cap = most < few ? most : few;
  return (int)(need < cap ? need : cap);
}

// any length: rows per share, about 2048 workgroups of 256 vectors each in all and no share of fewer than 8 rows
inline int64_t ln_bwd_chunk(int64_t rows, int c, int V) {
  const int cols = ((c + V - 1) / V + 255) / 256;
  const int64_t want = 2048 / cols + 1, most = (rows + 7) / 8, k = want < most ? want : most;
  return (rows + k - 1) / k;
}

inline int ln_bwd_shares(int64_t rows, int c, int pad, int V) {
  const int threads = ln_bwd_threads(rows, c, pad, V);
  if (threads) return ln_bwd_groups(rows, threads);
  const int64_t chunk = ln_bwd_chunk(rows, c, V);
  return (int)((rows + chunk - 1) / chunk);
}

// the most that a call of these rows leaves, whatever its type (V 4 or 8) and padding (which counts below one vector only)
inline int ln_bwd_most_shares(int64_t rows, int c) {
  int most = 0;
  for (int V = 4; V <= 8; V += 4)
    for (int pad = 0; pad <= V; pad += c < V ? V - c : V + 1) {
      const int n = ln_bwd_shares(rows, c, pad, V);
      if (n > most) most = n;
    }
  return most;
}

}  // namespace
