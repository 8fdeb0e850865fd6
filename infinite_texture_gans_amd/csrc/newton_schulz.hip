// Orthogonalisation by Newton-Schulz products, and the Muon optimiser step built on it (gfx950).
//
//   X = G / |G|_F (transposed so that its m rows are no more than its n columns), then per step
//   A = X X^T,   B = b A + c A A,   X <- a X + B X
//
// Arithmetic.  The products run on the fp16 matrix cores with fp32 accumulation.  X is carried as two fp16 planes hi + lo (22 bits):
// what a step rounds off X reappears in directions G does not have, and every later step multiplies it by a = 3.4 (X in fp16 alone:
// 8e-2 off for an update of rank 1), while what the products round off stays inside G's own row and column space.
// A and B are hi + lo as well and every product is hi hi + hi lo + lo hi: as near to 64 bits as fp32 products are, at three of the
// 16 MFMA issues an fp32 product of the same shape costs.  What is dropped is lo lo, 2^-22 of a product.  That holds for every type:
// a bf16 matrix is rounded once, at the end (one product of the hi planes would be off by 0.5 .. 1.5 of that rounding beside it, most
// where the matrix is small).
// The planes hold X * 2^12, A * 2^12 and B * 2^10, so that lo is a normal number wherever it matters; the spectral bound of X under
// the coefficients (checked on the host) keeps hi finite.
//
// All matrices of a call share one sequence of launches (norm, conversion, three per step): a launch covers the tiles of every
// matrix.  Planes are padded with zeros to whole tiles; zeros stay zeros under the iteration, so no product needs a mask.
#include <math.h>
#include "itg_common.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr float SX = 4096.f, SA = 4096.f, SB = 1024.f;
constexpr int NORM_ELEMS = 16384, NORM_BLOCKS = 512;      // values per partial sum of squares (at least), partial sums per matrix (at most)
constexpr int KSHARE = 256, KLONG = 1024;                 // a tile's K is split into shares of KSHARE or more, from KLONG on

// the three products of a step, the last of which writes the result after the last step
enum { PH_A = 0, PH_B = 1, PH_X = 2, PH_LAST = 3 };

struct NsMat {                 // one job: `count` matrices of the same shape
  int m, n, mp, np;            // short and long side, and their padded extents
  int count, tall, nblk;       // tall: the matrix has more rows than columns (X is its transpose)
  int norm0, conv0;            // first workgroup of this job in the launches
  int tile0[3], share0[3], shares[3], cut[3];      // per product (A, B, X): first tile, first share, shares of a split tile, split tiles
  int block0, blocks, subs;    // short sides: first workgroup, workgroups per matrix, column blocks per workgroup
  float scale;                 // muon: sqrt(max(1, rows / cols))
  int64_t in, ldi, sti, out, ldo, sto;      // element offsets, row strides, matrix strides
  int64_t ws, wst;             // bytes: first matrix's workspace, stride between matrices
};

struct NsArgs {
  NsMat j[ITG_NS_MAX_JOBS];
  int n, nesterov;
  int direct[3];               // per product: tiles that one workgroup does whole; those behind them are split along K
  char* ws; float* slab;       // slab: the split tiles' shares
  const void* g; void* out; float* mom; float* ema;
  float eps, mu, lr, wd, ema_decay;
};

// a matrix's workspace: double norm2[NORM_BLOCKS] | X planes (two generations) | A | B planes
struct NsWs {
  double* part;
  _Float16* x[2][2];                  // [generation][hi, lo]: [mp][np]
  _Float16 *a[2], *b[2];              // [hi, lo]: [mp][mp]
};

__host__ __device__ inline int64_t ns_ws_bytes(int mp, int np) {
  const int64_t x = (int64_t)mp * np * 2, a = (int64_t)mp * mp * 2;
  return (int64_t)NORM_BLOCKS * 8 + 4 * x + 4 * a;
}

__device__ inline NsWs ns_ws(char* base, int mp, int np) {
  NsWs w;
  const int64_t x = (int64_t)mp * np, a = (int64_t)mp * mp;
  w.part = (double*)base;
  _Float16* q = (_Float16*)(base + (int64_t)NORM_BLOCKS * 8);
  for (int g = 0; g < 2; ++g) {
    w.x[g][0] = q; q += x;
    w.x[g][1] = q; q += x;
  }
  w.a[0] = q; q += a;
  w.a[1] = q; q += a;
  w.b[0] = q; q += a;
  w.b[1] = q;
  return w;
}

// the job that owns workgroup `bid` of a launch; first(j): the launch's first workgroup of job j
template <typename F>
__device__ __forceinline__ int ns_job(const NsArgs& p, int bid, F first) {
  int lo = 0, hi = p.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first(p.j[mid]) <= bid) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void split_f16(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };      // 16 bytes at the type's alignment

// what G is multiplied with, from the sum of its squares: 0 = a matrix without a direction; an infinity or a NaN in the matrix makes
// every value of it NaN
__device__ __forceinline__ double ns_scale(double sum, float eps) {
  const double norm = sqrt(sum);
  return norm <= (double)eps ? 0.0 : norm < INFINITY ? (double)SX / norm : (double)NAN;
}

// four values of the result (columns row0 .. + 3 of X's row `col`), or what the optimiser step makes of them
template <typename OUT, bool MUON>
__device__ __forceinline__ void ns_result(const NsArgs& p, const NsMat& j, int z, int row0, int col, const f32x4& v) {
  if (col >= j.m || row0 >= j.n) return;
  const int64_t o = j.out + z * j.sto + (j.tall ? (int64_t)row0 * j.ldo + col : (int64_t)col * j.ldo + row0), step = j.tall ? j.ldo : 1;
  OUT* out = (OUT*)p.out + o;
  const bool four = !j.tall && row0 + 4 <= j.n;        // four values side by side
  Pack<OUT, 4> old, res;
  Pack<float, 4> ema;
  if (MUON) {
    if (four) {
      old = *reinterpret_cast<const Pack<OUT, 4>*>(out);
      if (p.ema) ema = *reinterpret_cast<const Pack<float, 4>*>(p.ema + o);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (row0 + e < j.n) { old.v[e] = out[e * step]; if (p.ema) ema.v[e] = p.ema[o + e * step]; }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x = v[e] * (1.f / SX);
    if (MUON) {
      x = fmaf(-p.lr * j.scale, x, (float)old.v[e] * (1.f - p.lr * p.wd));
      ema.v[e] = fmaf(p.ema_decay, ema.v[e], (1.f - p.ema_decay) * x);
    }
    res.v[e] = (OUT)x;
  }
  if (four) {
    *reinterpret_cast<Pack<OUT, 4>*>(out) = res;
    if (MUON && p.ema) *reinterpret_cast<Pack<float, 4>*>(p.ema + o) = ema;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (row0 + e < j.n) { out[e * step] = res.v[e]; if (MUON && p.ema) p.ema[o + e * step] = ema.v[e]; }
  }
}

// ---- sum of squares (fp64: the range of fp32 gradients squared) in fixed shares; muon: the momentum is advanced here
template <typename T, bool MUON>
__global__ __launch_bounds__(1024) void ns_norm_kernel(NsArgs p) {
  constexpr int V = 16 / sizeof(T);
  const NsMat& j = p.j[ns_job(p, blockIdx.x, [](const NsMat& q) { return q.norm0; })];
  const int local = blockIdx.x - j.norm0, z = local / j.nblk, k = local - z * j.nblk;
  const int rows = j.tall ? j.n : j.m, cols = j.tall ? j.m : j.n;
  const int64_t total = (int64_t)rows * cols, per = ((total + j.nblk - 1) / j.nblk + V - 1) / V * V;
  const int64_t e0 = k * per, e1 = e0 + per < total ? e0 + per : total;
  const T* g = (const T*)p.g + j.in + z * j.sti;
  float* mom = MUON ? p.mom + j.in : nullptr;
  double s = 0.0;
  auto add = [&](float u) { s = fma((double)u, (double)u, s); };
  if (j.ldi == cols) {                      // one run of values
    for (int64_t e = e0 + (int64_t)threadIdx.x * V; e < e1; e += 1024 * V) {
      if (e + V <= e1) {
        const Pack<T, V> u = *reinterpret_cast<const Pack<T, V>*>(g + e);
        if (MUON) {
          Pack<float, V> m = *reinterpret_cast<const Pack<float, V>*>(mom + e);
#pragma unroll
          for (int q = 0; q < V; ++q) { m.v[q] = fmaf(p.mu, m.v[q], (float)u.v[q]); add(p.nesterov ? fmaf(p.mu, m.v[q], (float)u.v[q]) : m.v[q]); }
          *reinterpret_cast<Pack<float, V>*>(mom + e) = m;
        } else {
#pragma unroll
          for (int q = 0; q < V; ++q) add((float)u.v[q]);
        }
      } else {
        for (int64_t q = e; q < e1; ++q) {
          const float u = (float)g[q];
          if (MUON) {
            const float m = fmaf(p.mu, mom[q], u);
            mom[q] = m;
            add(p.nesterov ? fmaf(p.mu, m, u) : m);
          } else {
            add(u);
          }
        }
      }
    }
  } else {
    for (int64_t e = e0 + threadIdx.x; e < e1; e += 1024) { const int64_t r = e / cols; add((float)g[r * j.ldi + (e - r * cols)]); }
  }
  s = wave_sum_d(s);
  __shared__ double lds[16];
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double v = 0.0;
    for (int q = 0; q < 16; ++q) v += lds[q];
    ((double*)(p.ws + j.ws + z * j.wst))[k] = v;
  }
}

// ---- X = G / |G| as planes: 64 x 64 tiles of the padded matrix in G's own orientation, turned in LDS where G is tall
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ns_convert_kernel(NsArgs p) {
  const NsMat& j = p.j[ns_job(p, blockIdx.x, [](const NsMat& q) { return q.conv0; })];
  const int rp = j.tall ? j.np : j.mp, cp = j.tall ? j.mp : j.np;        // padded extents in G's orientation
  const int tc = cp / 64, per = tc * (rp / 64);
  int local = blockIdx.x - j.conv0;
  const int z = local / per;
  local -= z * per;
  const int r0 = local / tc * 64, c0 = local % tc * 64;
  const int rows = j.tall ? j.n : j.m, cols = j.tall ? j.m : j.n;
  const NsWs w = ns_ws(p.ws + j.ws + z * j.wst, j.mp, j.np);
  __shared__ double lds[4];
  __shared__ float tile[64][65];
  const int c = (threadIdx.x & 15) * 4, rt = threadIdx.x >> 4;
  const T* g = (const T*)p.g + j.in + z * j.sti;
  f32x4 v[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = r0 + rt + q * 16;
    const int64_t at = (int64_t)r * j.ldi + c0 + c;
    v[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r < rows && c0 + c + 4 <= cols) {
      const Pack<T, 4> u = *reinterpret_cast<const Pack<T, 4>*>(g + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[q][e] = (float)u.v[e];
      if (MUON) {
        const Pack<float, 4> m = *reinterpret_cast<const Pack<float, 4>*>(p.mom + j.in + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q][e] = p.nesterov ? fmaf(p.mu, m.v[e], v[q][e]) : m.v[e];
      }
    } else if (r < rows) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + c + e < cols) {
          v[q][e] = (float)g[at + e];
          if (MUON) v[q][e] = p.nesterov ? fmaf(p.mu, p.mom[j.in + at + e], v[q][e]) : p.mom[j.in + at + e];
        }
    }
  }
  double s = 0.0;
  for (int k = threadIdx.x; k < j.nblk; k += 256) s += w.part[k];
  s = wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  const double inv = ns_scale((lds[0] + lds[1]) + (lds[2] + lds[3]), p.eps);
  if (!j.tall) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t at = (int64_t)(r0 + rt + q * 16) * cp + c0 + c;
      f16x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) { _Float16 h, l; split_f16(inv == 0.0 ? 0.f : (float)((double)v[q][e] * inv), h, l); hi[e] = h; lo[e] = l; }
      *reinterpret_cast<f16x4*>(w.x[0][0] + at) = hi;
      *reinterpret_cast<f16x4*>(w.x[0][1] + at) = lo;
    }
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[rt + q * 16][c + e] = inv == 0.0 ? 0.f : (float)((double)v[q][e] * inv);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = rt + q * 16;
    const int64_t at = (int64_t)(c0 + r) * rp + r0 + c;
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) { _Float16 h, l; split_f16(tile[c + e][r], h, l); hi[e] = h; lo[e] = l; }
    *reinterpret_cast<f16x4*>(w.x[0][0] + at) = hi;
    *reinterpret_cast<f16x4*>(w.x[0][1] + at) = lo;
  }
}

// ---- the products: D[row][col] = sum_k P[row][k] Q[col][k] over T x T tiles, both operands K-contiguous
//
// Staging: 16-byte chunks go from global memory straight into LDS.  A wave's 64 lanes fill 1 KiB in lane order, so the chunk a
// lane FETCHES is permuted instead: chunk c of row r sits in slot c ^ f(r), which spreads the 16 rows an MFMA operand read
// touches over all banks (4 chunks a row, f = r / 2).
constexpr int BK = 32;                 // K of a slice: that of one MFMA
__device__ __forceinline__ int slot(int r, int c) { return c ^ ((r >> 1) & 3); }

// Product X takes its first operand, whose rows are X's COLUMNS, from X itself: slices of BK rows of X, T columns wide, read by the
// transposing LDS read (16 lanes give four rows of 16 columns, lane l gets column l).  A copy of X^T instead would be half of all
// bytes that product X moves.  The 16 rows a read touches are spread over the banks: rows of 128 bytes (T 64) lie on alternating
// halves of the banks, longer ones all on the same.
template <int T> __device__ __forceinline__ int slot_t(int r, int c) {
  return T == 64 ? c ^ (((r >> 1) & 1) * 2 + ((r >> 3) & 1) * 4) : c ^ (2 * ((r & 3) | ((r >> 1) & 4)));
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// columns .. + 15 of the 8 rows from `at` on (pitch T): what a lane of a fragment holds
template <int T> __device__ __forceinline__ f16x8 frag_t(const _Float16* at) {
  typedef __attribute__((address_space(3))) s16x4* P;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(const_cast<_Float16*>(at))), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(const_cast<_Float16*>(at + 4 * T)));
  const f16x4 u = __builtin_bit_cast(f16x4, a), v = __builtin_bit_cast(f16x4, b);
  return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
}

// T: tile, TR x T where TALL; WR x WC waves share it, each with FR x FC fragments of 16 x 16
template <int T_, bool TALL = false> struct Tile {
  static constexpr int T = T_, TR = TALL ? 2 * T_ : T_, WR = 2, WC = 2, WAVES = WR * WC, NT = WAVES * 64;
  static constexpr int FR = TR / WR / 16, FC = T / WC / 16;
  static constexpr int PP = TR * BK, PQ = T * BK, BUF = 2 * (PP + PQ);      // halves: a plane of each operand, one buffer
  static constexpr int LP = PP * 2 / 1024 / WAVES, LQ = PQ * 2 / 1024 / WAVES;      // loads of a wave per plane
};

template <typename C>
struct Acc { f32x4 v[C::FR][C::FC]; };

template <typename C>
__device__ __forceinline__ void acc_zero(Acc<C>& a) {
#pragma unroll
  for (int i = 0; i < C::FR; ++i)
#pragma unroll
    for (int k = 0; k < C::FC; ++k) a.v[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// DEPTH LDS buffers: DEPTH - 1 slices of K are on their way while one is multiplied
// acc = the product over k0 .. k1 (multiples of BK) of the T rows from P[plane] and Q[plane] on
// TURN: P[plane] holds the operand by column (row k of it at k * ldp)
template <typename C, int DEPTH, bool TURN>
__device__ __forceinline__ void ns_product(Acc<C>& acc, const _Float16* const* P, int ldp, const _Float16* const* Q, int ldq, int k0, int k1, _Float16* lds) {
  constexpr int T = C::T, TR = C::TR, CH = BK / 8, ROWS = 64 / CH, CHT = TR / 8, ROWST = 64 / CHT;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l15 = lane & 15, lk = lane >> 4;
  uint32_t from_p[C::LP], from_q[C::LQ];                   // bytes from a slice's first value to what this lane fetches
#pragma unroll
  for (int u = 0; u < C::LP; ++u) {
    const int r = (wave * C::LP + u) * ROWS + lane / CH, rt = (wave * C::LP + u) * ROWST + lane / CHT;
    from_p[u] = TURN ? (uint32_t)(rt * ldp + slot_t<TR>(rt, lane % CHT) * 8) * 2u : (uint32_t)(r * ldp + slot(r, lane % CH) * 8) * 2u;
  }
#pragma unroll
  for (int u = 0; u < C::LQ; ++u) {
    const int r = (wave * C::LQ + u) * ROWS + lane / CH;
    from_q[u] = (uint32_t)(r * ldq + slot(r, lane % CH) * 8) * 2u;
  }
  auto stage = [&](int buf, int k) {
    auto fetch = [&](const _Float16* from, const uint32_t* off, int n, _Float16* to) {
#pragma unroll
      for (int u = 0; u < n; ++u)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((const char*)from + off[u]),
                                         (__attribute__((address_space(3))) void*)(to + u * 512), 16, 0, 0);
    };
#pragma unroll
    for (int q = 0; q < 2; ++q)
      fetch(TURN ? P[q] + (int64_t)k * ldp : P[q] + k, from_p, C::LP, lds + buf * C::BUF + q * C::PP + wave * C::LP * 512);
#pragma unroll
    for (int q = 0; q < 2; ++q) fetch(Q[q] + k, from_q, C::LQ, lds + buf * C::BUF + 2 * C::PP + q * C::PQ + wave * C::LQ * 512);
  };
  const int wr = (wave / C::WC) * (TR / C::WR), wc = (wave % C::WC) * (T / C::WC);
  const int row_q = (wc + l15) * BK;
  const int ch = slot(l15, lk) * 8;
  int at_p[C::FR];
#pragma unroll
  for (int i = 0; i < C::FR; ++i) {
    const int r = lk * 8 + (l15 >> 2);
    at_p[i] = TURN ? r * TR + slot_t<TR>(r, wr / 8 + 2 * i + ((l15 >> 1) & 1)) * 8 + (l15 & 1) * 4 : (wr + i * 16 + l15) * BK;
  }
  // sums in two levels, a fresh accumulator every 256 of K.  One accumulator over all of K drifts: each MFMA adds to it
  // with an error of one step of the sum, and on the diagonal of X X^T, a sum of squares, these do not cancel (a 1 x 4099 matrix:
  // 2.9e-6 off with one level, fp32 products in torch 6e-7)
  constexpr int FLUSH = KSHARE / BK;
  Acc<C> part;
  acc_zero(acc);
  acc_zero(part);
  const int nk = (k1 - k0) / BK;
  constexpr int LOADS = 2 * (C::LP + C::LQ);               // of a wave per buffer
  struct Frags { f16x8 p[2][C::FR], q[2][C::FC]; };
  auto read = [&](int buf, Frags& f) {
    const _Float16* at = lds + buf * C::BUF;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int i = 0; i < C::FR; ++i)
        f.p[q][i] = TURN ? frag_t<TR>(at + q * C::PP + at_p[i]) : *reinterpret_cast<const f16x8*>(at + q * C::PP + at_p[i] + ch);
#pragma unroll
      for (int k = 0; k < C::FC; ++k) f.q[q][k] = *reinterpret_cast<const f16x8*>(at + 2 * C::PP + q * C::PQ + row_q + ch + k * 16 * BK);
    }
  };
  // lo hi, hi lo, hi hi: each over all fragments, so that no product waits for the one before it
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int q = 0; q < 3; ++q)
#pragma unroll
      for (int i = 0; i < C::FR; ++i)
#pragma unroll
        for (int k = 0; k < C::FC; ++k)
          part.v[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.p[q == 0][i], f.q[q == 1][k], part.v[i][k], 0, 0, 0);
  };
  auto flush = [&](int kk) {
    if ((kk + 1) % FLUSH != 0 && kk + 1 != nk) return;
#pragma unroll
    for (int i = 0; i < C::FR; ++i)
#pragma unroll
      for (int k = 0; k < C::FC; ++k) { acc.v[i][k] += part.v[i][k]; part.v[i][k] = f32x4{0.f, 0.f, 0.f, 0.f}; }
  };
  auto slice = [&](int k) { return k0 + (k < nk ? k : nk - 1) * BK; };      // past the end: the last slice again, so that the counts stay
  // A buffer has arrived when this wave's loads have (its own count: those of the buffers behind it may be in flight) and, by the
  // barrier, the other waves'.  The barrier also tells that the buffer before has been read and may be filled again.
  if (DEPTH == 4) {
    // few workgroups: nothing else hides the LDS reads, so a slice is read while the one before is multiplied
    Frags f[2];
#pragma unroll
    for (int b = 0; b < DEPTH; ++b) stage(b, slice(b));
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((DEPTH - 1) * LOADS) : "memory");
    read(0, f[0]);
    auto turn = [&](int kk, const Frags& now, Frags& next) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((DEPTH - 2) * LOADS) : "memory");
      stage(kk & 3, slice(kk + DEPTH));
      read((kk + 1) & 3, next);
      multiply(now);
      flush(kk);
    };
    int kk = 0;
    for (; kk + 1 < nk; kk += 2) { turn(kk, f[0], f[1]); turn(kk + 1, f[1], f[0]); }
    if (kk < nk) turn(kk, f[0], f[1]);
  } else {
#pragma unroll
    for (int b = 0; b < DEPTH - 1; ++b) stage(b, slice(b));
    int buf = 0, into = DEPTH - 1;
    for (int kk = 0; kk < nk; ++kk) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((DEPTH - 2) * LOADS) : "memory");
      stage(into, slice(kk + DEPTH - 1));
      Frags f;
      read(buf, f);
      multiply(f);
      flush(kk);
      buf = buf + 1 == DEPTH ? 0 : buf + 1;
      into = into + 1 == DEPTH ? 0 : into + 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // no load into LDS outlives the workgroup
}

// halves of LDS a wave needs to turn N x FC fragments into rows of 16-byte stores
template <int N, int FC> constexpr int ns_turn() { return FC * 16 * (N * 16 + 8) > N * 16 * (FC * 16 + 8) ? FC * 16 * (N * 16 + 8) : N * 16 * (FC * 16 + 8); }

// N x FC fragments (a lane: rows 4 lk .. + 3 of column l15) to dst, the address of the first row and column, through this wave's own
// LDS: as [row][column] or, BYCOL, as [column][row].  Rows of 32 halves and more leave in 16-byte stores; straight from the
// fragments they would be stores of 8 and of 2 bytes, in pieces of 32.
template <int N, int FC, bool BYCOL>
__device__ __forceinline__ void ns_store(_Float16* turn, const f16x4 (&v)[N][FC], _Float16* dst, int64_t ld) {
  constexpr int ROWS = BYCOL ? FC * 16 : N * 16, LEN = BYCOL ? N * 16 : FC * 16, PITCH = LEN + 8, CH = LEN / 8;
  const int lane = threadIdx.x & 63, l15 = lane & 15, lk = lane >> 4;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int k = 0; k < FC; ++k) {
      if (BYCOL) {
        *reinterpret_cast<f16x4*>(turn + (k * 16 + l15) * PITCH + i * 16 + lk * 4) = v[i][k];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) turn[(i * 16 + lk * 4 + e) * PITCH + k * 16 + l15] = v[i][k][e];
      }
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the wave's own writes, read by its other lanes
#pragma unroll
  for (int q = 0; q < ROWS * CH / 64; ++q) {
    const int id = q * 64 + lane, r = id / CH, c = id % CH * 8;
    *reinterpret_cast<f16x8*>(dst + (int64_t)r * ld + c) = *reinterpret_cast<const f16x8*>(turn + r * PITCH + c);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // read before the next call writes
}

// The operand whose tile a product's result is added to: A (product B) or X (product X), hi and lo.
template <typename C, int PH, int N>
struct Addend {
  f16x4 h[N][C::FC], l[N][C::FC];
  __device__ __forceinline__ void load(const NsMat& j, const NsWs& w, int ti, int tj, int gen, int i0) {
    if (PH == PH_A) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int rbase = ti * C::TR + (wave / C::WC) * (C::TR / C::WR) + i0 * 16 + (lane >> 4) * 4, cbase = tj * C::T + (wave % C::WC) * (C::T / C::WC) + (lane & 15);
    const _Float16* hi = PH == PH_B ? w.a[0] : w.x[gen][0];
    const _Float16* lo = PH == PH_B ? w.a[1] : w.x[gen][1];
    const int64_t ld = PH == PH_B ? j.mp : j.np;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < C::FC; ++k) {
        const int64_t at = (cbase + k * 16) * ld + rbase + i * 16;
        h[i][k] = *reinterpret_cast<const f16x4*>(hi + at);
        l[i][k] = *reinterpret_cast<const f16x4*>(lo + at);
      }
  }
};

// What a product's tile (ti, tj) of a matrix becomes; N fragment rows of it, from i0 on.  A lane holds rows row0 .. row0 + 3 of
// column col of each fragment.  The addend is read before the first store: loads and stores share one counter, so a load behind a
// store waits for it (reading fragment by fragment cost 15 us a tile).
template <typename C, int PH, typename OUT, bool MUON, int N>
__device__ __forceinline__ void ns_write_rows(const f32x4 (*acc)[C::FC], int i0, const Addend<C, PH, N>& ad, _Float16* lds, const NsArgs& p,
                                              const NsMat& j, const NsWs& w, int z, int ti, int tj, int gen, float ca, float cb, float cc) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l15 = lane & 15, lk = lane >> 4;
  const int r0 = ti * C::TR + (wave / C::WC) * (C::TR / C::WR) + i0 * 16, c0 = tj * C::T + (wave % C::WC) * (C::T / C::WC);
  f16x4 hi[N][C::FC], lo[N][C::FC];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int k = 0; k < C::FC; ++k) {
      const int row0 = r0 + i * 16 + lk * 4, col = c0 + k * 16 + l15;
      const f32x4 sum = acc[i][k];
      f32x4 v;
      if (PH == PH_A) {
        v = sum * (SA / (SX * SX));
      } else if (PH == PH_B) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a1 = (float)ad.h[i][k][e] * (1.f / SA) + (float)ad.l[i][k][e] * (1.f / SA), a2 = sum[e] * (1.f / (SA * SA));
          v[e] = (cb * a1 + cc * a2) * SB;
        }
      } else {      // row: column of X, col: row of X
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(ca, (float)ad.h[i][k][e] + (float)ad.l[i][k][e], sum[e] * (1.f / SB));
      }
      if (PH == PH_LAST) {
        ns_result<OUT, MUON>(p, j, z, row0, col, v);
        continue;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) { _Float16 h, l; split_f16(v[e], h, l); hi[i][k][e] = h; lo[i][k][e] = l; }
    }
  if (PH == PH_LAST) return;
  _Float16* turn = lds + wave * ns_turn<N, C::FC>();
  if (PH < PH_X) {
    _Float16* th = PH == PH_A ? w.a[0] : w.b[0];
    _Float16* tl = PH == PH_A ? w.a[1] : w.b[1];
    const int64_t down = (int64_t)c0 * j.mp + r0, across = (int64_t)r0 * j.mp + c0;
    ns_store<N, C::FC, true>(turn, hi, th + down, j.mp);
    ns_store<N, C::FC, true>(turn, lo, tl + down, j.mp);
    if (ti != tj) {
      ns_store<N, C::FC, false>(turn, hi, th + across, j.mp);
      ns_store<N, C::FC, false>(turn, lo, tl + across, j.mp);
    }
  } else {
    const int64_t at = (int64_t)c0 * j.np + r0;
    ns_store<N, C::FC, true>(turn, hi, w.x[gen ^ 1][0] + at, j.np);
    ns_store<N, C::FC, true>(turn, lo, w.x[gen ^ 1][1] + at, j.np);
  }
}

// matrix z and tile (ti, tj) of tile `local` of a job
template <int T, int TR, int PH>
__device__ __forceinline__ void ns_tile(const NsMat& j, int local, int& z, int& ti, int& tj) {
  const int nt = j.mp / T;
  if (PH >= PH_X) {
    const int per = nt * (j.np / TR);
    z = local / per; local -= z * per;
    // rows: X's columns, columns: X's rows.  Bands of 8 tile rows: the tiles a die works on at a time form a square, which reads
    // the fewest operand rows
    const int nr = j.np / TR, band = local / (8 * nt), in = local - band * 8 * nt, high = nr - band * 8 < 8 ? nr - band * 8 : 8;
    tj = in / high; ti = band * 8 + (in - tj * high);
  } else {
    const int per = nt * (nt + 1) / 2;
    z = local / per; local -= z * per;
    ti = 0;
    while (local >= nt - ti) { local -= nt - ti; ++ti; }
    tj = ti + local;                                     // upper triangle: the product is symmetric
  }
}

// One workgroup per tile, or, of the tiles behind direct[], per share of a tile's K, which goes to the slab: the tiles of a small
// call do not fill the chip, and neither do those that are left over from its last full round.
template <int T, bool TALL, int DEPTH, int PH, typename OUT, bool MUON>
__global__ __launch_bounds__((Tile<T>::NT), 2) void ns_gemm_kernel(NsArgs p, int gen, float ca, float cb, float cc) {
  typedef Tile<T, TALL> C;
  constexpr int Q3 = PH < PH_X ? PH : 2;
  extern __shared__ __attribute__((aligned(16))) _Float16 lds[];
  const int direct = p.direct[Q3], bid = blockIdx.x;
  const bool whole = bid < direct;
  int job, tile, share = 0, slot_at = 0;
  if (whole) {
    // neighbouring workgroups go to different dies (8, each with an L2 of its own): give each die a run of neighbouring tiles
    const int run = direct >> 3;
    const int t = bid < run * 8 ? (bid & 7) * run + (bid >> 3) : bid;
    job = ns_job(p, t, [](const NsMat& q) { return q.tile0[Q3]; });
    tile = t - p.j[job].tile0[Q3];
  } else {
    // the shares of a slice of K side by side, and on one die: they read the same operands
    slot_at = bid - direct;
    const int run = ((int)gridDim.x - direct) >> 3;
    if (slot_at < run * 8) slot_at = (slot_at & 7) * run + (slot_at >> 3);
    job = ns_job(p, slot_at, [](const NsMat& q) { return q.share0[Q3]; });
    const int at = slot_at - p.j[job].share0[Q3], n = p.j[job].cut[Q3];
    share = at / n;
    tile = at - share * n;
    if (p.j[job].tile0[Q3] < direct) tile += direct - p.j[job].tile0[Q3];
  }
  const NsMat& j = p.j[job];
  int z, ti, tj;
  ns_tile<T, C::TR, PH>(j, tile, z, ti, tj);
  const NsWs w = ns_ws(p.ws + j.ws + z * j.wst, j.mp, j.np);
  const int ld = PH == PH_A ? j.np : j.mp;                 // of the second operand, and K
  const _Float16* P[2]; const _Float16* Q[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    P[q] = PH >= PH_X ? w.x[gen][q] + ti * C::TR : (PH == PH_A ? w.x[gen][q] : w.a[q]) + (int64_t)ti * T * ld;
    Q[q] = (PH == PH_A ? w.x[gen][q] : PH == PH_B ? w.a[q] : w.b[q]) + (int64_t)tj * T * ld;
  }
  int k0 = 0, k1 = ld;
  if (!whole) {
    const int per = (ld + j.shares[Q3] * 64 - 1) / (j.shares[Q3] * 64) * 64;      // shares are multiples of 64
    k0 = share * per;
    k1 = k0 + per < ld ? k0 + per : ld;
  }
  // 64: the addend waits in registers through the product; larger tiles read it behind it, in halves
  constexpr int N = 2;
  Acc<C> acc;
  Addend<C, PH, N> ad;
  if (C::FR == N && whole) ad.load(j, w, ti, tj, gen, 0);
  ns_product<C, DEPTH, (PH >= PH_X)>(acc, P, PH >= PH_X ? j.np : ld, Q, ld, k0, k1, lds);
  if (whole) {
    if (C::FR != N) ad.load(j, w, ti, tj, gen, 0);
    __syncthreads();                                       // the slices in LDS have been read: it turns the results now
    ns_write_rows<C, PH, OUT, MUON, N>(acc.v, 0, ad, lds, p, j, w, z, ti, tj, gen, ca, cb, cc);
    if (C::FR > N) {
      ad.load(j, w, ti, tj, gen, N);
      ns_write_rows<C, PH, OUT, MUON, N>(acc.v + C::FR - N, N, ad, lds, p, j, w, z, ti, tj, gen, ca, cb, cc);
    }
  } else {
    f32x4* to = reinterpret_cast<f32x4*>(p.slab) + (int64_t)slot_at * (C::TR * T / 4) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < C::FR; ++i)
#pragma unroll
      for (int k = 0; k < C::FC; ++k) to[(i * C::FC + k) * C::NT] = acc.v[i][k];
  }
}

// the split tiles: their shares added in order, then as any other tile; a workgroup per row of fragments
template <int T, bool TALL, int PH, typename OUT, bool MUON>
__global__ __launch_bounds__((Tile<T>::NT)) void ns_join_kernel(NsArgs p, int gen, float ca, float cb, float cc) {
  typedef Tile<T, TALL> C;
  constexpr int Q3 = PH < PH_X ? PH : 2;
  const int direct = p.direct[Q3], t = direct + blockIdx.x / C::FR, i = blockIdx.x % C::FR;
  const NsMat& j = p.j[ns_job(p, t, [](const NsMat& q) { return q.tile0[Q3]; })];
  const int first = j.tile0[Q3] > direct ? j.tile0[Q3] : direct, n = j.shares[Q3];
  const f32x4* from = reinterpret_cast<const f32x4*>(p.slab) + (int64_t)(j.share0[Q3] + t - first) * (C::TR * T / 4) + i * C::FC * C::NT + threadIdx.x;
  const int64_t next = (int64_t)j.cut[Q3] * (C::TR * T / 4);
  __shared__ __attribute__((aligned(16))) _Float16 lds[C::WAVES * ns_turn<1, C::FC>()];
  int z, ti, tj;
  ns_tile<T, C::TR, PH>(j, t - j.tile0[Q3], z, ti, tj);
  const NsWs w = ns_ws(p.ws + j.ws + z * j.wst, j.mp, j.np);
  Addend<C, PH, 1> ad;
  ad.load(j, w, ti, tj, gen, i);
  f32x4 v[1][C::FC];
#pragma unroll
  for (int k = 0; k < C::FC; ++k) v[0][k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < n; ++s)
#pragma unroll
    for (int k = 0; k < C::FC; ++k) v[0][k] += from[s * next + k * C::NT];
  ns_write_rows<C, PH, OUT, MUON, 1>(v, i, ad, lds, p, j, w, z, ti, tj, gen, ca, cb, cc);
}

#include "newton_schulz_thin.h"

// ---- host side
// launches of a call: workgroups of norm and conversion; per product its tile size (TR: columns of X in a tile of product X), workgroups (whole tiles and shares) and split tiles
// thin: 0, or the short side that newton_schulz_thin.h holds; blocks: its workgroups; one: a matrix is one block
struct NsPlan { int64_t bytes, norm, conv; int T[3], TR; int64_t grid[3], join[3]; int thin; int64_t blocks; bool one; };

inline int64_t up(int64_t v, int64_t k) { return (v + k - 1) / k * k; }

// Tile sizes of the products, from the number of tiles that each size would make.
// X: 128 from 384 tiles on (1024 x 8192 fp32, 512 tiles: 820 -> 712 us a call; 1024 x 4096, 256 tiles: 508 -> 566).  Below, 64, as
//   tiles of 128 columns of X by 64 rows where they make 512 or more: a third less of LDS and cache traffic for a product (the default
//   generator's matrices, a Muon step: 417 -> 392 us; 2048 x 2048 835 -> 811; 512 x 4096, 256 such tiles: 217 -> 246).
// A and B, whose leftover tiles are split along K, go by tiles x K: 128 from 192 K on (1024 x 8192, A 288 K: 712 -> 673 us;
//   4 x 1024 x 1024, 144 K: 634 -> 642).
// A size whose padding adds more than an eighth to the planes is not taken (the default generator's matrices of 3 to 416 rows: 448 us
// a Muon step with X at 128, 430 without).
void ns_tile_sizes(const NsArgs& p, NsPlan& pl) {
  int64_t a = 0, b = 0, x = 0, x64 = 0, tall = 0;
  for (int i = 0; i < p.n; ++i) {
    const NsMat& j = p.j[i];
    const int64_t m = up(j.m, 128) / 128, n = up(j.n, 128) / 128, sym = m * (m + 1) / 2 * j.count;
    a += sym * n * 128;
    b += sym * m * 128;
    x += m * n * j.count;
    tall += up(j.m, 64) / 64 * n * j.count;
    x64 += up(j.m, 64) / 64 * (up(j.n, 64) / 64) * j.count;
  }
  const int64_t least = 192 * 1024;
  const bool fits = 32 * x <= 9 * x64;
  pl.T[0] = fits && a >= least ? 128 : 64;
  pl.T[1] = fits && b >= least ? 128 : 64;
  pl.T[2] = fits && x >= 384 ? 128 : 64;
  pl.TR = pl.T[2] == 64 && 16 * tall <= 9 * x64 && tall >= 512 ? 128 : pl.T[2];
}

// Tiles and shares of product q (A, B, X).  `slots` workgroups run at a time; whole rounds of them take a tile each, and what is
// left over is split along K until it fills a round of its own, in shares of no less than KSHARE.
int ns_tiles(NsArgs& p, NsPlan& pl, int q, int64_t& slab) {
  const int T = pl.T[q];
  int64_t tiles = 0;
  for (int i = 0; i < p.n; ++i) {
    NsMat& j = p.j[i];
    const int64_t nt = j.mp / T, nx = j.np / pl.TR;
    j.tile0[q] = (int)tiles;
    tiles += (q == 2 ? nt * nx : nt * (nt + 1) / 2) * j.count;
    if (tiles >= ((int64_t)1 << 24)) return ITG_ERR_ARG;
  }
  const int64_t slots = 512;
  int64_t direct = tiles / slots * slots, rest = tiles - direct, shares = 0;
  // more than half a round left, or nothing to split: the last round stays as it is
  bool splits = false;
  for (int i = 0; i < p.n; ++i) splits |= (q == 0 ? p.j[i].np : p.j[i].mp) >= KLONG;
  if (!splits || rest * 2 > slots) { direct = tiles; rest = 0; }
  if (rest) {
    for (int64_t per = KSHARE;; per += KSHARE) {           // the shortest shares that fit one round
      shares = 0;
      for (int i = 0; i < p.n; ++i) {
        NsMat& j = p.j[i];
        const int64_t end = i + 1 < p.n ? p.j[i + 1].tile0[q] : tiles, first = j.tile0[q] > direct ? j.tile0[q] : direct;
        const int K = q == 0 ? j.np : j.mp;
        j.share0[q] = (int)shares;
        j.shares[q] = (int)((K + per - 1) / per);
        j.cut[q] = (int)(end > first ? end - first : 0);
        shares += (int64_t)j.cut[q] * j.shares[q];
      }
      if (shares <= slots || per >= ITG_NS_MAX_DIM) break;
    }
  }
  p.direct[q] = (int)direct;
  pl.grid[q] = direct + shares;
  pl.join[q] = rest;
  const int64_t each = (int64_t)(q == 2 ? pl.TR : T) * T * 4;
  if (shares * each > slab) slab = shares * each;
  return ITG_OK;
}

void ns_job_fields(const itg_ns_job& q, NsMat& j) {
  const int64_t blocks = ((int64_t)j.m * j.n + NORM_ELEMS - 1) / NORM_ELEMS;
  j.nblk = (int)(blocks < NORM_BLOCKS ? blocks : NORM_BLOCKS);
  j.scale = sqrtf(fmaxf(1.f, (float)q.rows / (float)q.cols));
  j.in = q.in_offset; j.ldi = q.in_ld; j.sti = q.in_stride;
  j.out = q.out_offset; j.ldo = q.out_ld; j.sto = q.out_stride;
}

// Short sides: every matrix of the call has at most 64 rows or columns, or 128, and its blocks of 128 columns make no more workgroups
// than a workgroup can add up shares of A in passing: 16 KiB each at 64, 32 of them with up to 4 blocks a workgroup (64 x 8192 fp32:
// 99 us, general path 129), 64 KiB at 128, 8 of them (128 x 1024: 116 us against 122; 128 x 2048 in 16: 140 against 127).
bool ns_thin(NsArgs& p, NsPlan& pl) {
  int m = 0, n = 0;
  for (int i = 0; i < p.n; ++i) { m = p.j[i].m > m ? p.j[i].m : m; n = p.j[i].n > n ? p.j[i].n : n; }
  if (m > 128) return false;
  const int M = m > 64 ? 128 : 64, most = M == 64 ? 32 : 8, turns = M == 64 ? 4 : 1;
  if (up(n, 128) / 128 > most * turns) return false;
  pl.thin = M;
  pl.one = n <= 128;
  for (int i = 0; i < p.n; ++i) {
    NsMat& j = p.j[i];
    const int cols = (int)(up(j.n, 128) / 128);
    j.subs = (cols + most - 1) / most;
    j.blocks = (cols + j.subs - 1) / j.subs;
  }
  return true;
}

// fills p.j[] from the jobs; returns a status
int ns_plan(const itg_ns_job* jobs, int n, bool muon, NsArgs& p, NsPlan& pl) {
  if (!jobs || n < 1 || n > ITG_NS_MAX_JOBS) return ITG_ERR_ARG;
  p.n = n;
  pl = NsPlan{};
  for (int i = 0; i < n; ++i) {
    const itg_ns_job& q = jobs[i];
    if (q.rows < 1 || q.cols < 1 || q.rows > ITG_NS_MAX_DIM || q.cols > ITG_NS_MAX_DIM || q.count < 1 || q.reserved) return ITG_ERR_ARG;
    if (q.in_offset < 0 || q.out_offset < 0 || q.in_ld < q.cols || q.out_ld < q.cols || q.in_stride < 0 || q.out_stride < 0) return ITG_ERR_ARG;
    const int64_t most = (int64_t)1 << 60;      // no offset of the call passes 63 bits
    if (q.in_ld > most / q.rows || q.out_ld > most / q.rows || q.in_stride > most / q.count || q.out_stride > most / q.count ||
        q.in_offset > most || q.out_offset > most) return ITG_ERR_ARG;
    if (muon && (q.count != 1 || q.in_ld != q.cols || q.out_ld != q.cols || q.in_offset != q.out_offset)) return ITG_ERR_ARG;
    if (muon)
      for (int k = 0; k < i; ++k) {
        const int64_t o = jobs[k].out_offset;
        if (q.out_offset < o + (int64_t)jobs[k].rows * jobs[k].cols && o < q.out_offset + (int64_t)q.rows * q.cols) return ITG_ERR_ARG;
      }
    if (q.count > 1 && q.out_stride < (int64_t)(q.rows - 1) * q.out_ld + q.cols) return ITG_ERR_ARG;      // results may not overlap
    NsMat& j = p.j[i];
    j.tall = q.rows > q.cols;
    j.m = j.tall ? q.cols : q.rows; j.n = j.tall ? q.rows : q.cols;
    j.count = q.count;
  }
  if (ns_thin(p, pl)) {
    for (int i = 0; i < n; ++i) {
      const itg_ns_job& q = jobs[i];
      NsMat& j = p.j[i];
      j.mp = pl.thin; j.np = (int)up(j.n, 128);
      ns_job_fields(q, j);
      j.norm0 = (int)pl.norm; j.block0 = (int)pl.blocks;
      pl.norm += (int64_t)j.nblk * j.count;
      pl.blocks += (int64_t)j.blocks * j.count;
      // a launch counts its threads in 32 bits
      if ((!pl.one && pl.norm >= ((int64_t)1 << 22)) || pl.blocks * 4 * pl.thin >= ((int64_t)1 << 32)) return ITG_ERR_ARG;
      j.wst = pl.one ? 0 : up(thin_ws_bytes(pl.thin, j.np, j.blocks), 256);
      j.ws = pl.bytes;
      if (j.wst > ((int64_t)1 << 60) / j.count) return ITG_ERR_ARG;
      pl.bytes += j.wst * j.count;
    }
    if (pl.one) pl.bytes = 16;
    return ITG_OK;
  }
  ns_tile_sizes(p, pl);
  const int T = pl.T[2] > pl.T[0] ? pl.T[2] : pl.T[0] > pl.T[1] ? pl.T[0] : pl.T[1];
  for (int i = 0; i < n; ++i) {
    const itg_ns_job& q = jobs[i];
    NsMat& j = p.j[i];
    j.mp = (int)up(j.m, T); j.np = (int)up(j.n, T > pl.TR ? T : pl.TR);
    ns_job_fields(q, j);
    j.norm0 = (int)pl.norm; j.conv0 = (int)pl.conv;
    pl.norm += (int64_t)j.nblk * j.count;
    pl.conv += (int64_t)(j.mp / 64) * (j.np / 64) * j.count;
    if (pl.norm >= ((int64_t)1 << 22) || pl.conv >= ((int64_t)1 << 24)) return ITG_ERR_ARG;      // a launch counts its threads in 32 bits
    j.wst = up(ns_ws_bytes(j.mp, j.np), 256);
    j.ws = pl.bytes;
    if (j.wst > ((int64_t)1 << 60) / j.count) return ITG_ERR_ARG;
    pl.bytes += j.wst * j.count;
  }
  int64_t slab = 0;
  for (int q = 0; q < 3; ++q) {
    const int rc = ns_tiles(p, pl, q, slab);
    if (rc) return rc;
  }
  p.slab = (float*)pl.bytes;      // an offset until the call has its workspace
  pl.bytes += slab;
  return ITG_OK;
}

// The planes hold |X| < 16, |A| < 16 and |B| < 64: every step's polynomial has to keep X's singular values below 3.9 and the
// spectrum of B below 60 on the interval its predecessors leave (the first one's is [0, 1]).
bool ns_coefficients_ok(const float* abc, int steps) {
  double top = 1.0;
  for (int s = 0; s < steps; ++s, abc += 3) {
    const double a = abc[0], b = abc[1], c = abc[2];
    if (!isfinite(a) || !isfinite(b) || !isfinite(c)) return false;
    double next = 0.0;
    for (int i = 0; i <= 128; ++i) {
      const double x = top * i / 128.0, q = x * x, poly = q * (b + c * q), y = fabs(x * (a + poly));
      if (!(fabs(poly) <= 60.0) || !(y <= 3.9)) return false;
      if (y > next) next = y;
    }
    top = next;
  }
  return true;
}

template <typename K>
int ns_lds(K kernel, int bytes) {
  return bytes <= 64 * 1024 || hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess
             ? ITG_OK : ITG_ERR_LAUNCH;
}

template <int T, int DEPTH, int PH, typename OUT, bool MUON, bool TALL = false>
int ns_launch(const NsArgs& p, const NsPlan& pl, int gen, const float* abc, hipStream_t s) {
  typedef Tile<T, TALL> C;
  constexpr int Q3 = PH < PH_X ? PH : 2, LDS = DEPTH * C::BUF * 2;
  if (ns_lds(&ns_gemm_kernel<T, TALL, DEPTH, PH, OUT, MUON>, LDS)) return ITG_ERR_LAUNCH;
  hipLaunchKernelGGL((ns_gemm_kernel<T, TALL, DEPTH, PH, OUT, MUON>), dim3((unsigned)pl.grid[Q3]), dim3(C::NT), LDS, s, p, gen, abc[0], abc[1], abc[2]);
  ITG_CHECK_LAUNCH();
  if (pl.join[Q3]) {
    hipLaunchKernelGGL((ns_join_kernel<T, TALL, PH, OUT, MUON>), dim3((unsigned)(pl.join[Q3] * C::FR)), dim3(C::NT), 0, s, p, gen, abc[0], abc[1], abc[2]);
    ITG_CHECK_LAUNCH();
  }
  return ITG_OK;
}

template <int PH, typename OUT, bool MUON>
int ns_phase(const NsArgs& p, const NsPlan& pl, int gen, const float* abc, hipStream_t s) {
  const int T = pl.T[PH < PH_X ? PH : 2];
  const int64_t grid = pl.grid[PH < PH_X ? PH : 2];
  // 64: four buffers while two workgroups a CU take the whole launch (512 x 512: 156 us against 182 with two,
  // 2 x 1501 x 333: 185 against 196), two buffers and up to five workgroups a CU beyond
  if (PH >= PH_X && T == 64 && pl.TR == 128) return ns_launch<64, 2, PH, OUT, MUON, (PH >= PH_X)>(p, pl, gen, abc, s);
  if (T == 64 && grid <= 512) return ns_launch<64, 4, PH, OUT, MUON>(p, pl, gen, abc, s);
  if (T == 64) return ns_launch<64, 2, PH, OUT, MUON>(p, pl, gen, abc, s);
  return ns_launch<128, 2, PH, OUT, MUON>(p, pl, gen, abc, s);
}

template <int M, typename T, bool MUON>
int ns_thin_run(const NsArgs& p, const NsPlan& pl, const float* abc, int steps, hipStream_t s) {
  typedef Thin<M> C;
  const dim3 grid((unsigned)pl.blocks), nt(C::NT);
  if (pl.one) {
    NsSteps st;
    for (int i = 0; i < 3 * steps; ++i) st.abc[i] = abc[i];
    st.n = steps;
    if (ns_lds(&ns_thin_all_kernel<M, T, MUON>, C::LDS)) return ITG_ERR_LAUNCH;
    hipLaunchKernelGGL((ns_thin_all_kernel<M, T, MUON>), grid, nt, C::LDS, s, p, st);
    ITG_CHECK_LAUNCH();
    return ITG_OK;
  }
  if (ns_lds(&ns_thin_first_kernel<M, T, MUON>, C::LDS) || ns_lds(&ns_thin_step_kernel<M, false, T, MUON>, C::LDS) ||
      ns_lds(&ns_thin_step_kernel<M, true, T, MUON>, C::LDS)) return ITG_ERR_LAUNCH;
  hipLaunchKernelGGL((ns_norm_kernel<T, MUON>), dim3((unsigned)pl.norm), dim3(1024), 0, s, p);
  ITG_CHECK_LAUNCH();
  hipLaunchKernelGGL((ns_thin_first_kernel<M, T, MUON>), grid, nt, C::LDS, s, p);
  ITG_CHECK_LAUNCH();
  for (int k = 0; k < steps; ++k, abc += 3) {
    if (k + 1 < steps) hipLaunchKernelGGL((ns_thin_step_kernel<M, false, T, MUON>), grid, nt, C::LDS, s, p, k & 1, abc[0], abc[1], abc[2]);
    else hipLaunchKernelGGL((ns_thin_step_kernel<M, true, T, MUON>), grid, nt, C::LDS, s, p, k & 1, abc[0], abc[1], abc[2]);
    ITG_CHECK_LAUNCH();
  }
  return ITG_OK;
}

template <typename T, bool MUON>
int ns_run(NsArgs& p, const NsPlan& pl, const float* abc, int steps, hipStream_t s) {
  if (pl.thin) return pl.thin == 64 ? ns_thin_run<64, T, MUON>(p, pl, abc, steps, s) : ns_thin_run<128, T, MUON>(p, pl, abc, steps, s);
  p.slab = (float*)(p.ws + (int64_t)p.slab);
  hipLaunchKernelGGL((ns_norm_kernel<T, MUON>), dim3((unsigned)pl.norm), dim3(1024), 0, s, p);
  ITG_CHECK_LAUNCH();
  hipLaunchKernelGGL((ns_convert_kernel<T, MUON>), dim3((unsigned)pl.conv), dim3(256), 0, s, p);
  ITG_CHECK_LAUNCH();
  for (int k = 0; k < steps; ++k, abc += 3) {
    const int gen = k & 1;
    int rc = ns_phase<PH_A, T, MUON>(p, pl, gen, abc, s);
    if (!rc) rc = ns_phase<PH_B, T, MUON>(p, pl, gen, abc, s);
    if (!rc) rc = k + 1 < steps ? ns_phase<PH_X, T, MUON>(p, pl, gen, abc, s) : ns_phase<PH_LAST, T, MUON>(p, pl, gen, abc, s);
    if (rc) return rc;
  }
  return ITG_OK;
}

// whether two matrices of different buffers share a value
bool muon_overlap(const itg_ns_job* jobs, int n, const float* const (&buf)[4]) {
  int64_t lo = jobs[0].out_offset, hi = lo;
  auto size = [](const itg_ns_job& j) { return (int64_t)j.rows * j.cols; };
  for (int i = 0; i < n; ++i) {
    lo = jobs[i].out_offset < lo ? jobs[i].out_offset : lo;
    hi = jobs[i].out_offset + size(jobs[i]) > hi ? jobs[i].out_offset + size(jobs[i]) : hi;
  }
  for (int a = 0; a < 4; ++a)
    for (int b = 0; b < a; ++b) {
      if (!buf[a] || !buf[b]) continue;
      const int64_t apart = (int64_t)((uintptr_t)buf[a] - (uintptr_t)buf[b]);      // bytes from a value of b to a's
      if (apart >= (hi - lo) * 4 || -apart >= (hi - lo) * 4) continue;
      for (int i = 0; i < n; ++i)
        for (int k = 0; k < n; ++k) {
          const int64_t from = apart + (jobs[i].out_offset - jobs[k].out_offset) * 4;
          if (from < size(jobs[k]) * 4 && -from < size(jobs[i]) * 4) return true;
        }
    }
  return false;
}

}  // namespace

extern "C" {

int64_t itg_newton_schulz_workspace(const itg_ns_job* jobs, int n, int dtype) {
  if (dtype < ITG_F32 || dtype > ITG_F16) return ITG_ERR_ARG;
  NsArgs p; NsPlan pl;
  const int rc = ns_plan(jobs, n, false, p, pl);
  return rc ? rc : pl.bytes;
}

int itg_newton_schulz(const itg_ns_job* jobs, int n, int dtype, const void* g, void* out, int steps, const float* coefficients,
                      float eps, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype < ITG_F32 || dtype > ITG_F16 || !g || !out || !coefficients || steps < 1 || steps > ITG_NS_MAX_STEPS || !(eps >= 0.f)) return ITG_ERR_ARG;
  if (((uintptr_t)g | (uintptr_t)out) & (dtype == ITG_F32 ? 3 : 1)) return ITG_ERR_ALIGN;
  NsArgs p; NsPlan pl;
  const int rc = ns_plan(jobs, n, false, p, pl);
  if (rc) return rc;
  if (!ns_coefficients_ok(coefficients, steps)) return ITG_ERR_ARG;
  if (!workspace || workspace_bytes < pl.bytes) return ITG_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return ITG_ERR_ALIGN;
  p.ws = (char*)workspace; p.g = g; p.out = out; p.mom = nullptr; p.ema = nullptr; p.eps = eps; p.nesterov = 0;
  p.mu = p.lr = p.wd = p.ema_decay = 0.f;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == ITG_F32) return ns_run<float, false>(p, pl, coefficients, steps, s);
  if (dtype == ITG_BF16) return ns_run<__bf16, false>(p, pl, coefficients, steps, s);
  return ns_run<_Float16, false>(p, pl, coefficients, steps, s);
}

int itg_muon_step(const itg_ns_job* jobs, int n, float* param, const float* g, float* momentum, float* ema, float lr, float mu,
                  int nesterov, float weight_decay, float ema_decay, int steps, const float* coefficients, float eps,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (!param || !g || !momentum || !coefficients || steps < 1 || steps > ITG_NS_MAX_STEPS || !(eps >= 0.f)) return ITG_ERR_ARG;
  if (param == g || param == momentum || g == momentum || ema == param || ema == g || ema == momentum) return ITG_ERR_ARG;
  if (((uintptr_t)param | (uintptr_t)g | (uintptr_t)momentum | (uintptr_t)ema) & 3) return ITG_ERR_ALIGN;
  NsArgs p; NsPlan pl;
  const int rc = ns_plan(jobs, n, true, p, pl);
  if (rc) return rc;
  const float* const buf[4] = {param, g, momentum, ema};
  if (muon_overlap(jobs, n, buf)) return ITG_ERR_ARG;
  if (!ns_coefficients_ok(coefficients, steps)) return ITG_ERR_ARG;
  if (!workspace || workspace_bytes < pl.bytes) return ITG_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return ITG_ERR_ALIGN;
  p.ws = (char*)workspace; p.g = g; p.out = param; p.mom = momentum; p.ema = ema; p.eps = eps; p.nesterov = nesterov ? 1 : 0;
  p.mu = mu; p.lr = lr; p.wd = weight_decay; p.ema_decay = ema_decay;
  return ns_run<float, true>(p, pl, coefficients, steps, (hipStream_t)stream);
}

}  // extern "C"
