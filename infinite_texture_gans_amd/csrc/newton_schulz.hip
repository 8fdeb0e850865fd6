// Orthogonalisation by Newton-Schulz products, and the Muon optimiser step built on it (gfx950).
//
//   X = G / |G|_F (transposed so that its m rows are no more than its n columns), then per step
//   A = X X^T,   B = b A + c A A,   X <- a X + B X
//
// Arithmetic.  The products run on the fp16 matrix cores with fp32 accumulation.  X is carried as two fp16 planes hi + lo (22 bits):
// what a step rounds off X reappears in directions G does not have, and every later step multiplies it by a = 3.4 (X in fp16 alone:
// 8e-2 off for an update of rank 1), while what the products round off stays inside G's own row and column space.
//   split (fp32 and fp16 matrices): A and B are hi + lo as well and every product is hi hi + hi lo + lo hi: as near to 64 bits as
//     fp32 products are, at three of the 16 MFMA issues an fp32 product of the same shape costs;
//   single (bf16 matrices): one product of the hi planes.  The diagonals of A and B, which are the large entries and whose rounding
//     would scale a whole row, stay fp32 (the planes hold zero there) and join in the epilogues: the error beside the result's own
//     rounding to bf16 stays at 0.6 of it or less.
// The planes hold X * 2^12, A * 2^12 and B * 2^10, so that lo is a normal number wherever it matters; the spectral bound of X under
// the coefficients (checked on the host) keeps hi finite.
//
// All matrices of a call share one sequence of launches (norm, conversion, three per step): a launch covers the tiles of every
// matrix.  Planes are padded with zeros to whole tiles; zeros stay zeros under the iteration, so no product needs a mask.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include "itg_common.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr float SX = 4096.f, SA = 4096.f, SB = 1024.f;
constexpr int NORM_ELEMS = 16384, NORM_BLOCKS = 512;      // elements per partial sum of squares, partial sums per matrix

struct NsMat {                 // one job: `count` matrices of the same shape
  int m, n, mp, np;            // short and long side, and their padded extents
  int count, tall, nblk;       // tall: the matrix has more rows than columns (X is its transpose)
  int norm0, conv0, sym0, x0;  // first workgroup of this job in the launches
  float scale;                 // muon: sqrt(max(1, rows / cols))
  int64_t in, ldi, sti, out, ldo, sto;      // element offsets, row strides, matrix strides
  int64_t ws, wst;             // bytes: first matrix's workspace, stride between matrices
};

struct NsArgs {
  NsMat j[ITG_NS_MAX_JOBS];
  int n, nesterov;
  char* ws;
  const void* g; void* out; float* mom; float* ema;
  float eps, mu, lr, wd, ema_decay;
};

// a matrix's workspace: double norm2[NORM_BLOCKS] | X, X^T planes (two generations) | A | B planes | their diagonals
struct NsWs {
  double* part;
  _Float16 *xr[2][2], *xt[2][2];      // [generation][hi, lo]: [mp][np] and [np][mp]
  _Float16 *a[2], *b[2];              // [hi, lo]: [mp][mp]
  float *da, *db;                     // diagonals of A and B (single)
};

__host__ __device__ inline int64_t ns_ws_bytes(int mp, int np, bool split) {
  const int64_t x = (int64_t)mp * np * 2, a = (int64_t)mp * mp * 2;
  return (int64_t)NORM_BLOCKS * 8 + 2 * x * (split ? 4 : 3) + a * (split ? 4 : 2) + (int64_t)mp * 8;
}

__device__ inline NsWs ns_ws(char* base, int mp, int np, bool split) {
  NsWs w;
  const int64_t x = (int64_t)mp * np, a = (int64_t)mp * mp;
  w.part = (double*)base;
  _Float16* q = (_Float16*)(base + (int64_t)NORM_BLOCKS * 8);
  for (int g = 0; g < 2; ++g) {
    w.xr[g][0] = q; q += x;
    w.xr[g][1] = q; q += x;
    w.xt[g][0] = q; q += x;
    w.xt[g][1] = q; q += split ? x : 0;
  }
  w.a[0] = q; q += a;
  w.a[1] = q; q += split ? a : 0;
  w.b[0] = q; q += a;
  w.b[1] = q; q += split ? a : 0;
  w.da = (float*)q; w.db = w.da + mp;
  return w;
}

// the job that owns workgroup `bid` of a launch; FIRST is the launch's offset field
template <int NsMat::*FIRST>
__device__ __forceinline__ int ns_job(const NsArgs& p, int bid) {
  int lo = 0, hi = p.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.j[mid].*FIRST <= bid) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void split_f16(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

template <typename T> __device__ __forceinline__ float ld_f(const T* q) { return (float)*q; }
template <> __device__ __forceinline__ float ld_f<__hip_bfloat16>(const __hip_bfloat16* q) { return __bfloat162float(*q); }
template <typename T> __device__ __forceinline__ void st_f(T* q, float v) { *q = (T)v; }
template <> __device__ __forceinline__ void st_f<__hip_bfloat16>(__hip_bfloat16* q, float v) { *q = __float2bfloat16(v); }

// ---- sum of squares (fp64: the range of fp32 gradients squared) in fixed shares; muon: the momentum is advanced here
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs p, bool split) {
  const NsMat& j = p.j[ns_job<&NsMat::norm0>(p, blockIdx.x)];
  const int local = blockIdx.x - j.norm0, z = local / j.nblk, k = local - z * j.nblk;
  const int rows = j.tall ? j.n : j.m, cols = j.tall ? j.m : j.n;
  const int64_t total = (int64_t)rows * cols, per = (total + j.nblk - 1) / j.nblk;
  const int64_t e0 = k * per, e1 = e0 + per < total ? e0 + per : total;
  const T* g = (const T*)p.g + j.in + z * j.sti;
  double s = 0.0;
  for (int64_t e = e0 + threadIdx.x; e < e1; e += 256) {
    const int64_t r = e / cols, at = r * j.ldi + (e - r * cols);
    float u = ld_f(g + at);
    if (MUON) {
      float* mom = p.mom + j.in + at;
      const float v = fmaf(p.mu, *mom, u);
      *mom = v;
      u = p.nesterov ? fmaf(p.mu, v, u) : v;
    }
    s += (double)u * (double)u;
  }
  s = wave_sum_d(s);
  __shared__ double lds[4];
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) ns_ws(p.ws + j.ws + z * j.wst, j.mp, j.np, split).part[k] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// ---- X = G / |G| as planes, both orientations: 64 x 64 tiles of the padded matrix in G's own orientation
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ns_convert_kernel(NsArgs p, bool split) {
  const NsMat& j = p.j[ns_job<&NsMat::conv0>(p, blockIdx.x)];
  const int rp = j.tall ? j.np : j.mp, cp = j.tall ? j.mp : j.np;        // padded extents in G's orientation
  const int tc = cp / 64, per = tc * (rp / 64);
  int local = blockIdx.x - j.conv0;
  const int z = local / per;
  local -= z * per;
  const int r0 = local / tc * 64, c0 = local % tc * 64;
  const int rows = j.tall ? j.n : j.m, cols = j.tall ? j.m : j.n;
  const NsWs w = ns_ws(p.ws + j.ws + z * j.wst, j.mp, j.np, split);
  __shared__ double lds[4];
  __shared__ float tile[64][65];
  double s = 0.0;
  for (int k = threadIdx.x; k < j.nblk; k += 256) s += w.part[k];
  s = wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt((lds[0] + lds[1]) + (lds[2] + lds[3]));
  // an infinity or a NaN in the matrix makes every value of it NaN
  const double inv = norm <= (double)p.eps ? 0.0 : norm < INFINITY ? (double)SX / norm : (double)NAN;
  const T* g = (const T*)p.g + j.in + z * j.sti;
  _Float16* nh = j.tall ? w.xt[0][0] : w.xr[0][0];
  _Float16* nl = j.tall ? w.xt[0][1] : w.xr[0][1];
  _Float16* oh = j.tall ? w.xr[0][0] : w.xt[0][0];
  _Float16* ol = j.tall ? w.xr[0][1] : w.xt[0][1];
  const bool keep_nl = split || !j.tall, keep_ol = split || j.tall;        // single: lo beside X only, not beside X^T
  const int c = threadIdx.x & 63;
  for (int r = threadIdx.x >> 6; r < 64; r += 4) {
    float v = 0.f;
    if (r0 + r < rows && c0 + c < cols) {
      const int64_t at = (int64_t)(r0 + r) * j.ldi + c0 + c;
      v = ld_f(g + at);
      if (MUON) {
        const float mv = p.mom[j.in + at];
        v = p.nesterov ? fmaf(p.mu, mv, v) : mv;
      }
      v = inv == 0.0 ? 0.f : (float)((double)v * inv);
    }
    tile[r][c] = v;
    _Float16 hi, lo;
    split_f16(v, hi, lo);
    nh[(int64_t)(r0 + r) * cp + c0 + c] = hi;
    if (keep_nl) nl[(int64_t)(r0 + r) * cp + c0 + c] = lo;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 6; r < 64; r += 4) {
    _Float16 hi, lo;
    split_f16(tile[c][r], hi, lo);
    oh[(int64_t)(c0 + r) * rp + r0 + c] = hi;
    if (keep_ol) ol[(int64_t)(c0 + r) * rp + r0 + c] = lo;
  }
}

// ---- the three products of a step: D[row][col] = sum_k P[row][k] Q[col][k] over T x T tiles, both operands K-contiguous
enum { PH_A = 0, PH_B = 1, PH_X = 2, PH_LAST = 3 };

// Staging: 16-byte chunks go from global memory straight into LDS.  A wave's 64 lanes fill 1 KiB in lane order, so the chunk a
// lane FETCHES is permuted instead: chunk c of row r sits in slot c ^ f(r), which spreads the 16 rows an MFMA operand read
// touches over all banks (BK 64: 8 chunks a row, f = r; BK 32: 4 chunks a row, f = r / 2).
template <int BK> __device__ __forceinline__ int slot(int r, int c) { return BK == 64 ? c ^ (r & 7) : c ^ ((r >> 1) & 3); }

template <int T, int BK>
__device__ __forceinline__ void stage(_Float16* lds, const _Float16* src, int64_t ld, int k0) {
  constexpr int CH = BK / 8, ROWS = 64 / CH;             // chunks per row, rows per wave load
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane / CH, pos = lane % CH;
#pragma unroll
  for (int q = wave; q < T / ROWS; q += 4) {
    const int row = q * ROWS + r;
    const _Float16* src_l = src + (int64_t)row * ld + k0 + slot<BK>(row, pos) * 8;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src_l,
                                     (__attribute__((address_space(3))) void*)(lds + q * ROWS * BK), 16, 0, 0);
  }
}

template <int T, int BK>
__device__ __forceinline__ f16x8 frag(const _Float16* lds, int row, int chunk) {
  return *reinterpret_cast<const f16x8*>(lds + row * BK + slot<BK>(row, chunk) * 8);
}

template <int T, bool SPLIT, int PH, typename OUT, bool MUON>
__global__ __launch_bounds__(256) void ns_gemm_kernel(NsArgs p, int gen, float ca, float cb, float cc) {
  constexpr int BK = SPLIT ? 32 : 64, NP = SPLIT ? 2 : 1, F = T / 32;      // F x F fragments of 16 x 16 per wave
  __shared__ __attribute__((aligned(16))) _Float16 lds[2][2][NP][T * BK];  // [buffer][operand][plane]
  const NsMat& j = p.j[PH >= PH_X ? ns_job<&NsMat::x0>(p, blockIdx.x) : ns_job<&NsMat::sym0>(p, blockIdx.x)];
  int local = blockIdx.x - (PH >= PH_X ? j.x0 : j.sym0), z, ti, tj;
  const int nt = j.mp / T;
  if (PH >= PH_X) {
    const int per = nt * (j.np / T);
    z = local / per; local -= z * per;
    ti = local / nt; tj = local - ti * nt;               // rows: X's columns, columns: X's rows
  } else {
    const int per = nt * (nt + 1) / 2;
    z = local / per; local -= z * per;
    ti = 0;
    while (local >= nt - ti) { local -= nt - ti; ++ti; }
    tj = ti + local;                                     // upper triangle: the product is symmetric
  }
  const NsWs w = ns_ws(p.ws + j.ws + z * j.wst, j.mp, j.np, SPLIT);
  const int64_t ld = PH == PH_A ? j.np : j.mp;
  const int K = (int)ld;
  const _Float16* P[2]; const _Float16* Q[2];
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    P[q] = (PH == PH_A ? w.xr[gen][q] : PH == PH_B ? w.a[q] : w.xt[gen][q]) + (int64_t)ti * T * ld;
    Q[q] = (PH == PH_A ? w.xr[gen][q] : PH == PH_B ? w.a[q] : w.b[q]) + (int64_t)tj * T * ld;
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l15 = lane & 15, lk = lane >> 4;
  const int wr = (wave >> 1) * (T / 2), wc = (wave & 1) * (T / 2);
  f32x4 acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int k = 0; k < F; ++k) acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
  // split: sums in two levels, a fresh accumulator every 256 of K.  One accumulator over all of K drifts: each MFMA adds to it
  // with an error of one step of the sum, and on the diagonal of X X^T, a sum of squares, these do not cancel (a 1 x 4099 matrix:
  // 2.9e-6 off with one level, fp32 products in torch 6e-7)
  constexpr int FLUSH = 256 / BK;
  f32x4 sum[SPLIT ? F : 1][SPLIT ? F : 1];
  if (SPLIT) {
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int k = 0; k < F; ++k) sum[SPLIT ? i : 0][SPLIT ? k : 0] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int nk = K / BK;
#pragma unroll
  for (int q = 0; q < NP; ++q) { stage<T, BK>(lds[0][0][q], P[q], ld, 0); stage<T, BK>(lds[0][1][q], Q[q], ld, 0); }
  for (int kk = 0; kk < nk; ++kk) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // this buffer's chunks have arrived (mine; the barrier covers the others')
    __syncthreads();
    const int cur = kk & 1;
    if (kk + 1 < nk) {
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        stage<T, BK>(lds[cur ^ 1][0][q], P[q], ld, (kk + 1) * BK);
        stage<T, BK>(lds[cur ^ 1][1][q], Q[q], ld, (kk + 1) * BK);
      }
    }
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      f16x8 fp[NP][F], fq[NP][F];
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int i = 0; i < F; ++i) {
          fp[q][i] = frag<T, BK>(lds[cur][0][q], wr + i * 16 + l15, ks * 4 + lk);
          fq[q][i] = frag<T, BK>(lds[cur][1][q], wc + i * 16 + l15, ks * 4 + lk);
        }
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int k = 0; k < F; ++k) {
          if (SPLIT) {
            acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[NP - 1][i], fq[0][k], acc[i][k], 0, 0, 0);
            acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[0][i], fq[NP - 1][k], acc[i][k], 0, 0, 0);
          }
          acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[0][i], fq[0][k], acc[i][k], 0, 0, 0);
        }
    }
    if (SPLIT && ((kk + 1) % FLUSH == 0 || kk + 1 == nk)) {
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int k = 0; k < F; ++k) { sum[SPLIT ? i : 0][SPLIT ? k : 0] += acc[i][k]; acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f}; }
    }
  }
  if (SPLIT) {
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int k = 0; k < F; ++k) acc[i][k] = sum[SPLIT ? i : 0][SPLIT ? k : 0];
  }
  // a lane holds rows row0 .. row0 + 3 of column col of each fragment
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int k = 0; k < F; ++k) {
      const int row0 = ti * T + wr + i * 16 + lk * 4, col = tj * T + wc + k * 16 + l15;
      f16x4 hi, lo;
      if (PH < PH_X) {
        f32x4 v;
        if (PH == PH_A) {
          v = acc[i][k] * (SA / (SX * SX));
        } else {
          const int64_t at = (int64_t)col * j.mp + row0;                    // A is symmetric: four consecutive values
          const f16x4 ah = *reinterpret_cast<const f16x4*>(w.a[0] + at);
          f16x4 al;
          if (SPLIT) al = *reinterpret_cast<const f16x4*>(w.a[1] + at);
          const float dcol = SPLIT ? 0.f : w.da[col];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a1 = (float)ah[e] * (1.f / SA), a2 = acc[i][k][e] * (1.f / (SA * SA));
            if (SPLIT) {
              a1 += (float)al[e] * (1.f / SA);
            } else {
              const float drow = w.da[row0 + e];
              if (row0 + e == col) { a1 = drow; a2 = fmaf(drow, drow, a2); }
              else a2 = fmaf(drow + dcol, a1, a2);
            }
            v[e] = (cb * a1 + cc * a2) * SB;
          }
        }
        if (!SPLIT) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (row0 + e == col) {
              if (PH == PH_A) w.da[col] = v[e] * (1.f / SA); else w.db[col] = v[e] * (1.f / SB);
              v[e] = 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) { _Float16 h, l; split_f16(v[e], h, l); hi[e] = h; lo[e] = l; }
        _Float16* oh = PH == PH_A ? w.a[0] : w.b[0];
        _Float16* ol = PH == PH_A ? w.a[1] : w.b[1];
        *reinterpret_cast<f16x4*>(oh + (int64_t)col * j.mp + row0) = hi;
        if (SPLIT) *reinterpret_cast<f16x4*>(ol + (int64_t)col * j.mp + row0) = lo;
        if (ti != tj) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            oh[(int64_t)(row0 + e) * j.mp + col] = hi[e];
            if (SPLIT) ol[(int64_t)(row0 + e) * j.mp + col] = lo[e];
          }
        }
      } else {
        // row: column of X, col: row of X
        const int64_t at = (int64_t)col * j.np + row0;
        const f16x4 xh = *reinterpret_cast<const f16x4*>(w.xr[gen][0] + at), xl = *reinterpret_cast<const f16x4*>(w.xr[gen][1] + at);
        const float dcol = SPLIT ? 0.f : w.db[col];
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = fmaf(ca, (float)xh[e] + (float)xl[e], acc[i][k][e] * (1.f / SB));
          if (!SPLIT) v[e] = fmaf(dcol, (float)xh[e], v[e]);
        }
        if (PH == PH_X) {
#pragma unroll
          for (int e = 0; e < 4; ++e) { _Float16 h, l; split_f16(v[e], h, l); hi[e] = h; lo[e] = l; }
          *reinterpret_cast<f16x4*>(w.xr[gen ^ 1][0] + at) = hi;
          *reinterpret_cast<f16x4*>(w.xr[gen ^ 1][1] + at) = lo;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w.xt[gen ^ 1][0][(int64_t)(row0 + e) * j.mp + col] = hi[e];
            if (SPLIT) w.xt[gen ^ 1][1][(int64_t)(row0 + e) * j.mp + col] = lo[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (row0 + e >= j.n || col >= j.m) continue;
            const float x = v[e] * (1.f / SX);
            const int64_t o = j.out + z * j.sto + (j.tall ? (int64_t)(row0 + e) * j.ldo + col : (int64_t)col * j.ldo + row0 + e);
            OUT* out = (OUT*)p.out + o;
            if (MUON) {
              const float q = fmaf(-p.lr * j.scale, x, ld_f(out) * (1.f - p.lr * p.wd));
              st_f(out, q);
              if (p.ema) p.ema[o] = fmaf(p.ema_decay, p.ema[o], (1.f - p.ema_decay) * q);
            } else {
              st_f(out, x);
            }
          }
        }
      }
    }
}

// ---- host side
struct NsPlan { int64_t bytes; int64_t norm, conv, sym, x; int T; };

inline int64_t up(int64_t v, int64_t k) { return (v + k - 1) / k * k; }

// fills p.j[] from the jobs; returns a status
int ns_plan(const itg_ns_job* jobs, int n, bool split, bool muon, NsArgs& p, NsPlan& pl) {
  if (!jobs || n < 1 || n > ITG_NS_MAX_JOBS) return ITG_ERR_ARG;
  p.n = n;
  pl = NsPlan{0, 0, 0, 0, 0, 64};
  for (int i = 0; i < n; ++i) {
    const itg_ns_job& q = jobs[i];
    if (q.rows < 1 || q.cols < 1 || q.rows > ITG_NS_MAX_DIM || q.cols > ITG_NS_MAX_DIM || q.count < 1 || q.reserved) return ITG_ERR_ARG;
    if (q.in_offset < 0 || q.out_offset < 0 || q.in_ld < q.cols || q.out_ld < q.cols || q.in_stride < 0 || q.out_stride < 0) return ITG_ERR_ARG;
    const int64_t most = (int64_t)1 << 60;      // no offset of the call passes 63 bits
    if (q.in_ld > most / q.rows || q.out_ld > most / q.rows || q.in_stride > most / q.count || q.out_stride > most / q.count ||
        q.in_offset > most || q.out_offset > most) return ITG_ERR_ARG;
    if (muon && (q.count != 1 || q.in_ld != q.cols || q.out_ld != q.cols || q.in_offset != q.out_offset)) return ITG_ERR_ARG;
    if (q.count > 1 && q.out_stride < (int64_t)(q.rows - 1) * q.out_ld + q.cols) return ITG_ERR_ARG;      // results may not overlap
    NsMat& j = p.j[i];
    j.tall = q.rows > q.cols;
    j.m = j.tall ? q.cols : q.rows; j.n = j.tall ? q.rows : q.cols;
    j.mp = (int)up(j.m, pl.T); j.np = (int)up(j.n, pl.T);
    j.count = q.count;
    const int64_t blocks = ((int64_t)j.m * j.n + NORM_ELEMS - 1) / NORM_ELEMS;
    j.nblk = (int)(blocks < NORM_BLOCKS ? blocks : NORM_BLOCKS);
    j.scale = sqrtf(fmaxf(1.f, (float)q.rows / (float)q.cols));
    j.in = q.in_offset; j.ldi = q.in_ld; j.sti = q.in_stride;
    j.out = q.out_offset; j.ldo = q.out_ld; j.sto = q.out_stride;
    const int64_t nt = j.mp / pl.T, nx = j.np / pl.T;
    j.norm0 = (int)pl.norm; j.conv0 = (int)pl.conv; j.sym0 = (int)pl.sym; j.x0 = (int)pl.x;
    pl.norm += (int64_t)j.nblk * j.count;
    pl.conv += (int64_t)(j.mp / 64) * (j.np / 64) * j.count;
    pl.sym += nt * (nt + 1) / 2 * j.count;
    pl.x += nt * nx * j.count;
    if (pl.norm > INT32_MAX || pl.conv > INT32_MAX || pl.sym > INT32_MAX || pl.x > INT32_MAX) return ITG_ERR_ARG;
    j.wst = up(ns_ws_bytes(j.mp, j.np, split), 256);
    j.ws = pl.bytes;
    if (j.wst > ((int64_t)1 << 60) / j.count) return ITG_ERR_ARG;
    pl.bytes += j.wst * j.count;
  }
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
    for (int i = 0; i <= 4096; ++i) {
      const double x = top * i / 4096.0, q = x * x, poly = q * (b + c * q), y = fabs(x * (a + poly));
      if (!(fabs(poly) <= 60.0) || !(y <= 3.9)) return false;
      if (y > next) next = y;
    }
    top = next;
  }
  return true;
}

template <typename T, bool SPLIT, bool MUON>
int ns_run(const NsArgs& p, const NsPlan& pl, const float* abc, int steps, hipStream_t s) {
  hipLaunchKernelGGL((ns_norm_kernel<T, MUON>), dim3((unsigned)pl.norm), dim3(256), 0, s, p, SPLIT);
  ITG_CHECK_LAUNCH();
  hipLaunchKernelGGL((ns_convert_kernel<T, MUON>), dim3((unsigned)pl.conv), dim3(256), 0, s, p, SPLIT);
  ITG_CHECK_LAUNCH();
  const dim3 sym((unsigned)pl.sym), x((unsigned)pl.x);
  for (int k = 0; k < steps; ++k, abc += 3) {
    const int gen = k & 1;
    hipLaunchKernelGGL((ns_gemm_kernel<64, SPLIT, PH_A, T, MUON>), sym, dim3(256), 0, s, p, gen, abc[0], abc[1], abc[2]);
    ITG_CHECK_LAUNCH();
    hipLaunchKernelGGL((ns_gemm_kernel<64, SPLIT, PH_B, T, MUON>), sym, dim3(256), 0, s, p, gen, abc[0], abc[1], abc[2]);
    ITG_CHECK_LAUNCH();
    if (k + 1 < steps)
      hipLaunchKernelGGL((ns_gemm_kernel<64, SPLIT, PH_X, T, MUON>), x, dim3(256), 0, s, p, gen, abc[0], abc[1], abc[2]);
    else
      hipLaunchKernelGGL((ns_gemm_kernel<64, SPLIT, PH_LAST, T, MUON>), x, dim3(256), 0, s, p, gen, abc[0], abc[1], abc[2]);
    ITG_CHECK_LAUNCH();
  }
  return ITG_OK;
}

}  // namespace

extern "C" {

int64_t itg_newton_schulz_workspace(const itg_ns_job* jobs, int n, int dtype) {
  if (dtype < ITG_F32 || dtype > ITG_F16) return ITG_ERR_ARG;
  NsArgs p; NsPlan pl;
  const int rc = ns_plan(jobs, n, dtype != ITG_BF16, false, p, pl);
  return rc ? rc : pl.bytes;
}

int itg_newton_schulz(const itg_ns_job* jobs, int n, int dtype, const void* g, void* out, int steps, const float* coefficients,
                      float eps, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype < ITG_F32 || dtype > ITG_F16 || !g || !out || !coefficients || steps < 1 || steps > ITG_NS_MAX_STEPS || !(eps >= 0.f)) return ITG_ERR_ARG;
  if (((uintptr_t)g | (uintptr_t)out) & (dtype == ITG_F32 ? 3 : 1)) return ITG_ERR_ALIGN;
  NsArgs p; NsPlan pl;
  const int rc = ns_plan(jobs, n, dtype != ITG_BF16, false, p, pl);
  if (rc) return rc;
  if (!ns_coefficients_ok(coefficients, steps)) return ITG_ERR_ARG;
  if (!workspace || workspace_bytes < pl.bytes) return ITG_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return ITG_ERR_ALIGN;
  p.ws = (char*)workspace; p.g = g; p.out = out; p.mom = nullptr; p.ema = nullptr; p.eps = eps; p.nesterov = 0;
  p.mu = p.lr = p.wd = p.ema_decay = 0.f;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == ITG_F32) return ns_run<float, true, false>(p, pl, coefficients, steps, s);
  if (dtype == ITG_BF16) return ns_run<__hip_bfloat16, false, false>(p, pl, coefficients, steps, s);
  return ns_run<_Float16, true, false>(p, pl, coefficients, steps, s);
}

int itg_muon_step(const itg_ns_job* jobs, int n, float* param, const float* g, float* momentum, float* ema, float lr, float mu,
                  int nesterov, float weight_decay, float ema_decay, int steps, const float* coefficients, float eps,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (!param || !g || !momentum || !coefficients || steps < 1 || steps > ITG_NS_MAX_STEPS || !(eps >= 0.f)) return ITG_ERR_ARG;
  if (((uintptr_t)param | (uintptr_t)g | (uintptr_t)momentum | (uintptr_t)ema) & 3) return ITG_ERR_ALIGN;
  NsArgs p; NsPlan pl;
  const int rc = ns_plan(jobs, n, true, true, p, pl);
  if (rc) return rc;
  if (!ns_coefficients_ok(coefficients, steps)) return ITG_ERR_ARG;
  if (!workspace || workspace_bytes < pl.bytes) return ITG_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return ITG_ERR_ALIGN;
  p.ws = (char*)workspace; p.g = g; p.out = param; p.mom = momentum; p.ema = ema; p.eps = eps; p.nesterov = nesterov ? 1 : 0;
  p.mu = mu; p.lr = lr; p.wd = weight_decay; p.ema_decay = ema_decay;
  return ns_run<float, true, true>(p, pl, coefficients, steps, (hipStream_t)stream);
}

}  // extern "C"
