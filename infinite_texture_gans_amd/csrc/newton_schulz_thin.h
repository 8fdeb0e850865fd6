// Matrices with a short side of at most M = 64 or 128: the whole iteration in one workgroup per matrix while the long side fits a
// block of 128 columns, and one launch per step beyond, in which every workgroup makes B for itself.  Included by newton_schulz.hip.
//
// A workgroup holds a block X[M][128] and A (then B) [M][M] in LDS, in rows padded by 8 halves: 16 rows read at the same column then
// start at 16 different groups of 4 banks.  A step is
//   A = X X^T (each wave a part of it), B = b A + c A A in A's place, X <- a X + B X in X's place (each wave its own columns, read by the
//   transposing LDS read), and with several blocks the shares of the next A go to the slab [blocks][M][M], which every workgroup of
//   the next step adds up in block order.
// What bounds it is latency: 16 matrices of 64 x 64 take 22 us in one launch, where the
// general path's 17 launches take 80.

template <int M> struct Thin {
  static constexpr int NW = M / 16, NT = NW * 64, W = 128, PX = W + 8, PA = M + 8;
  static constexpr int AR = 2, AC = M / 32, WAC = 2;               // A: fragments of a wave, waves side by side
  static constexpr int XR = W / NW / 16, XC = M / 16;              // X: a wave has XR * 16 columns of X and all rows
  static constexpr int LDS_X = 2 * M * PX, LDS_A = 2 * M * PA;    // halves
  static constexpr int LDS = (LDS_X + LDS_A) * 2 + 16 * 8;
  static constexpr int VEC = 8;                                    // vectors of 4 values of a block that a thread loads
};

template <int M> struct ThinLds {
  typedef Thin<M> C;
  _Float16 *x[2], *a[2];
  double* red;
  __device__ __forceinline__ explicit ThinLds(_Float16* lds) {
    x[0] = lds; x[1] = lds + M * C::PX;
    a[0] = lds + C::LDS_X; a[1] = a[0] + M * C::PA;
    red = (double*)(lds + C::LDS_X + C::LDS_A);
  }
};

// columns j0 .. j0 + 127 of G as X sees it, 4 values to a vector along G's rows; muon: with the momentum, advanced here if ADVANCE
template <typename C, int M, typename T, bool MUON, bool ADVANCE>
__device__ __forceinline__ void thin_load(const NsArgs& p, const NsMat& j, int z, int j0, f32x4 (&v)[C::VEC]) {
  const T* g = (const T*)p.g + j.in + z * j.sti;
  float* mom = MUON ? p.mom + j.in : nullptr;
#pragma unroll
  for (int q = 0; q < C::VEC; ++q) {
    const int id = q * C::NT + threadIdx.x;
    const int r = j.tall ? j0 + id / (M / 4) : id / (C::W / 4), c = j.tall ? id % (M / 4) * 4 : j0 + id % (C::W / 4) * 4;      // in G
    const int rows = j.tall ? j.n : j.m, cols = j.tall ? j.m : j.n;
    const int64_t at = r * j.ldi + c;
    v[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r >= rows) continue;
    if (c + 4 <= cols) {
      const Pack<T, 4> u = *reinterpret_cast<const Pack<T, 4>*>(g + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[q][e] = (float)u.v[e];
      if (MUON) {
        Pack<float, 4> m = *reinterpret_cast<const Pack<float, 4>*>(mom + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (ADVANCE) m.v[e] = fmaf(p.mu, m.v[e], v[q][e]);
          v[q][e] = p.nesterov ? fmaf(p.mu, m.v[e], v[q][e]) : m.v[e];
        }
        if (ADVANCE) *reinterpret_cast<Pack<float, 4>*>(mom + at) = m;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < cols) {
          float u = (float)g[at + e];
          if (MUON) {
            float m = mom[at + e];
            if (ADVANCE) { m = fmaf(p.mu, m, u); mom[at + e] = m; }
            u = p.nesterov ? fmaf(p.mu, m, u) : m;
          }
          v[q][e] = u;
        }
    }
  }
}

template <typename C, int M>
__device__ __forceinline__ void thin_put(const ThinLds<M>& s, bool tall, const f32x4 (&v)[C::VEC], double inv) {
#pragma unroll
  for (int q = 0; q < C::VEC; ++q) {
    const int id = q * C::NT + threadIdx.x;
    const int i = tall ? id % (M / 4) * 4 : id / (C::W / 4), j = tall ? id / (M / 4) : id % (C::W / 4) * 4;
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) { _Float16 h, l; split_f16(inv == 0.0 ? 0.f : (float)((double)v[q][e] * inv), h, l); hi[e] = h; lo[e] = l; }
    if (!tall) {
      *reinterpret_cast<f16x4*>(s.x[0] + i * C::PX + j) = hi;
      *reinterpret_cast<f16x4*>(s.x[1] + i * C::PX + j) = lo;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) { s.x[0][(i + e) * C::PX + j] = hi[e]; s.x[1][(i + e) * C::PX + j] = lo[e]; }
    }
  }
}

// acc += lo hi + hi lo + hi hi of fragments P[hi, lo][R] and Q[hi, lo][N]
template <int R, int N>
__device__ __forceinline__ void thin_mfma(f32x4 (&acc)[R][N], const f16x8 (&P)[2][R], const f16x8 (&Q)[2][N]) {
#pragma unroll
  for (int q = 0; q < 3; ++q)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(P[q == 0][i], Q[q == 1][k], acc[i][k], 0, 0, 0);
}

// this wave's part of S S^T over `slices` x 32 of the planes' columns (pitch PITCH), added to acc
template <typename C, int M, int PITCH>
__device__ __forceinline__ void thin_square(f32x4 (&acc)[C::AR][C::AC], _Float16* const* S, int slices) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l15 = lane & 15, lk = lane >> 4;
  const int wr = wave / C::WAC * (C::AR * 16), wc = wave % C::WAC * (C::AC * 16);
  f32x4 part[C::AR][C::AC];                                // a block's sum of its own (see ns_product)
#pragma unroll
  for (int i = 0; i < C::AR; ++i)
#pragma unroll
    for (int k = 0; k < C::AC; ++k) part[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int ks = 0; ks < slices; ++ks) {
    f16x8 P[2][C::AR], Q[2][C::AC];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int i = 0; i < C::AR; ++i) P[q][i] = *reinterpret_cast<const f16x8*>(S[q] + (wr + i * 16 + l15) * PITCH + ks * 32 + lk * 8);
#pragma unroll
      for (int k = 0; k < C::AC; ++k) Q[q][k] = *reinterpret_cast<const f16x8*>(S[q] + (wc + k * 16 + l15) * PITCH + ks * 32 + lk * 8);
    }
    thin_mfma<C::AR, C::AC>(part, P, Q);
  }
#pragma unroll
  for (int i = 0; i < C::AR; ++i)
#pragma unroll
    for (int k = 0; k < C::AC; ++k) acc[i][k] += part[i][k];
}

// A from its sum, then B in its place.  The caller has a barrier before (what lay there has been read), one is behind.
template <typename C, int M>
__device__ __forceinline__ void thin_poly(const ThinLds<M>& s, f32x4 (&acc)[C::AR][C::AC], float cb, float cc) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l15 = lane & 15, lk = lane >> 4;
  const int wr = wave / C::WAC * (C::AR * 16) + lk * 4, wc = wave % C::WAC * (C::AC * 16) + l15;
  auto put = [&](const f32x4& v, int row0, int col) {      // symmetric: four rows of a column are four of a row
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) { _Float16 h, l; split_f16(v[e], h, l); hi[e] = h; lo[e] = l; }
    *reinterpret_cast<f16x4*>(s.a[0] + col * C::PA + row0) = hi;
    *reinterpret_cast<f16x4*>(s.a[1] + col * C::PA + row0) = lo;
  };
#pragma unroll
  for (int i = 0; i < C::AR; ++i)
#pragma unroll
    for (int k = 0; k < C::AC; ++k) { put(acc[i][k] * (SA / (SX * SX)), wr + i * 16, wc + k * 16); acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __syncthreads();
  thin_square<C, M, C::PA>(acc, s.a, M / 32);
#pragma unroll
  for (int i = 0; i < C::AR; ++i)
#pragma unroll
    for (int k = 0; k < C::AC; ++k) {
      const int row0 = wr + i * 16, col = wc + k * 16;
      const f16x4 ah = *reinterpret_cast<const f16x4*>(s.a[0] + col * C::PA + row0), al = *reinterpret_cast<const f16x4*>(s.a[1] + col * C::PA + row0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a1 = (float)ah[e] * (1.f / SA) + (float)al[e] * (1.f / SA), a2 = acc[i][k][e] * (1.f / (SA * SA));
        acc[i][k][e] = (cb * a1 + cc * a2) * SB;
      }
    }
  __syncthreads();                                         // A has been read
#pragma unroll
  for (int i = 0; i < C::AR; ++i)
#pragma unroll
    for (int k = 0; k < C::AC; ++k) put(acc[i][k], wr + i * 16, wc + k * 16);
  __syncthreads();
}

// this wave's columns of the block: X <- a X + B X, in place, or the result
template <typename C, int M, bool LAST, typename OUT, bool MUON>
__device__ __forceinline__ void thin_update(const ThinLds<M>& s, const NsArgs& p, const NsMat& j, int z, int j0, float ca) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l15 = lane & 15, lk = lane >> 4, c0 = wave * C::XR * 16;
  if (j0 + c0 >= j.n) return;                              // zeros behind the matrix stay
  f32x4 acc[C::XR][C::XC];
#pragma unroll
  for (int i = 0; i < C::XR; ++i)
#pragma unroll
    for (int k = 0; k < C::XC; ++k) acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < M / 32; ++ks) {
    f16x8 P[2][C::XR], Q[2][C::XC];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int i = 0; i < C::XR; ++i) P[q][i] = frag_t<C::PX>(s.x[q] + (ks * 32 + lk * 8 + (l15 >> 2)) * C::PX + c0 + i * 16 + (l15 & 3) * 4);
#pragma unroll
      for (int k = 0; k < C::XC; ++k) Q[q][k] = *reinterpret_cast<const f16x8*>(s.a[q] + (k * 16 + l15) * C::PA + ks * 32 + lk * 8);
    }
    thin_mfma<C::XR, C::XC>(acc, P, Q);
  }
#pragma unroll
  for (int i = 0; i < C::XR; ++i)
#pragma unroll
    for (int k = 0; k < C::XC; ++k) {
      const int row0 = c0 + i * 16 + lk * 4, col = k * 16 + l15;
      _Float16 *xh = s.x[0] + col * C::PX + row0, *xl = s.x[1] + col * C::PX + row0;
      const f16x4 oh = *reinterpret_cast<const f16x4*>(xh), ol = *reinterpret_cast<const f16x4*>(xl);
      f32x4 v;
      f16x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = fmaf(ca, (float)oh[e] + (float)ol[e], acc[i][k][e] * (1.f / SB));
        _Float16 h, l;
        split_f16(v[e], h, l);
        hi[e] = h; lo[e] = l;
      }
      if (LAST) {
        ns_result<OUT, MUON>(p, j, z, j0 + row0, col, v);
      } else {
        *reinterpret_cast<f16x4*>(xh) = hi;
        *reinterpret_cast<f16x4*>(xl) = lo;
      }
    }
}

// ---- one launch: 1 / |G|, all steps, the result
struct NsSteps { float abc[3 * ITG_NS_MAX_STEPS]; int n; };

template <int M, typename T, bool MUON>
__global__ __launch_bounds__((Thin<M>::NT)) void ns_thin_all_kernel(NsArgs p, NsSteps st) {
  typedef Thin<M> C;
  extern __shared__ __attribute__((aligned(16))) _Float16 lds[];
  const ThinLds<M> s(lds);
  const NsMat& j = p.j[ns_job(p, blockIdx.x, [](const NsMat& q) { return q.block0; })];
  const int z = blockIdx.x - j.block0;
  f32x4 v[C::VEC];
  thin_load<C, M, T, MUON, true>(p, j, z, 0, v);
  double sum = 0.0;
#pragma unroll
  for (int q = 0; q < C::VEC; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = fma((double)v[q][e], (double)v[q][e], sum);
  sum = wave_sum_d(sum);
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int q = 0; q < C::NW; ++q) sum += s.red[q];
  thin_put<C, M>(s, j.tall, v, ns_scale(sum, p.eps));
  for (int k = 0; k < st.n; ++k) {
    __syncthreads();                                       // X is whole, B has been read
    f32x4 acc[C::AR][C::AC] = {};
    thin_square<C, M, C::PX>(acc, s.x, (j.n + 31) / 32);      // n <= 128: no more of the block than the matrix fills
    thin_poly<C, M>(s, acc, st.abc[3 * k + 1], st.abc[3 * k + 2]);
    if (k + 1 < st.n) thin_update<C, M, false, T, MUON>(s, p, j, z, 0, st.abc[3 * k]);
    else thin_update<C, M, true, T, MUON>(s, p, j, z, 0, st.abc[3 * k]);
  }
}

// ---- several blocks.  Workspace of a matrix: norm2[NORM_BLOCKS] | X hi | X lo [M][np] | slab [2][blocks][M * M]
__host__ __device__ inline int64_t thin_ws_bytes(int M, int np, int blocks) {
  return (int64_t)NORM_BLOCKS * 8 + (int64_t)2 * M * np * 2 + (int64_t)2 * blocks * M * M * 4;
}

struct ThinWs { double* part; _Float16* x[2]; float* slab[2]; };

__device__ __forceinline__ ThinWs thin_ws(char* base, int M, int np, int blocks) {
  ThinWs w;
  w.part = (double*)base;
  w.x[0] = (_Float16*)(base + (int64_t)NORM_BLOCKS * 8);
  w.x[1] = w.x[0] + (int64_t)M * np;
  w.slab[0] = (float*)(w.x[1] + (int64_t)M * np);
  w.slab[1] = w.slab[0] + (int64_t)blocks * M * M;
  return w;
}

// this wave's columns of the block from LDS to the planes
template <typename C, int M>
__device__ __forceinline__ void thin_keep(const ThinLds<M>& s, const ThinWs& w, int np, int j0) {
  constexpr int CH = C::XR * 2;                            // 16-byte chunks of a row
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the wave's own writes, read by its other lanes
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int u = 0; u < M * CH / 64; ++u) {
      const int id = u * 64 + lane, i = id / CH, c = wave * C::XR * 16 + id % CH * 8;
      *reinterpret_cast<f16x8*>(w.x[q] + (int64_t)i * np + j0 + c) = *reinterpret_cast<const f16x8*>(s.x[q] + i * C::PX + c);
    }
}

template <typename C>
__device__ __forceinline__ void thin_share(const f32x4 (&acc)[C::AR][C::AC], float* slab) {
  f32x4* to = reinterpret_cast<f32x4*>(slab) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < C::AR; ++i)
#pragma unroll
    for (int k = 0; k < C::AC; ++k) to[(i * C::AC + k) * C::NT] = acc[i][k];
}

// the planes of X and the shares of the first A
template <int M, typename T, bool MUON>
__global__ __launch_bounds__((Thin<M>::NT)) void ns_thin_first_kernel(NsArgs p) {
  typedef Thin<M> C;
  extern __shared__ __attribute__((aligned(16))) _Float16 lds[];
  const ThinLds<M> s(lds);
  const NsMat& j = p.j[ns_job(p, blockIdx.x, [](const NsMat& q) { return q.block0; })];
  const int local = blockIdx.x - j.block0, z = local / j.blocks, b = local - z * j.blocks;
  const ThinWs w = thin_ws(p.ws + j.ws + z * j.wst, M, j.np, j.blocks);
  const int first = b * j.subs * C::W, end = first + j.subs * C::W < j.np ? first + j.subs * C::W : j.np;
  f32x4 v[C::VEC];
  thin_load<C, M, T, MUON, false>(p, j, z, first, v);
  double sum = 0.0;
  for (int k = threadIdx.x; k < j.nblk; k += C::NT) sum += w.part[k];
  sum = wave_sum_d(sum);
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int q = 0; q < C::NW; ++q) sum += s.red[q];
  const double inv = ns_scale(sum, p.eps);
  f32x4 acc[C::AR][C::AC] = {};
  for (int j0 = first; j0 < end; j0 += C::W) {
    if (j0 != first) { thin_load<C, M, T, MUON, false>(p, j, z, j0, v); __syncthreads(); }      // the block before has been read
    thin_put<C, M>(s, j.tall, v, inv);
    __syncthreads();
    thin_keep<C, M>(s, w, j.np, j0);
    thin_square<C, M, C::PX>(acc, s.x, C::W / 32);
  }
  thin_share<C>(acc, w.slab[0] + (int64_t)b * M * M);
}

template <int M, bool LAST, typename T, bool MUON>
__global__ __launch_bounds__((Thin<M>::NT)) void ns_thin_step_kernel(NsArgs p, int gen, float ca, float cb, float cc) {
  typedef Thin<M> C;
  extern __shared__ __attribute__((aligned(16))) _Float16 lds[];
  const ThinLds<M> s(lds);
  const NsMat& j = p.j[ns_job(p, blockIdx.x, [](const NsMat& q) { return q.block0; })];
  const int local = blockIdx.x - j.block0, z = local / j.blocks, b = local - z * j.blocks;
  const ThinWs w = thin_ws(p.ws + j.ws + z * j.wst, M, j.np, j.blocks);
  const int first = b * j.subs * C::W, end = first + j.subs * C::W < j.np ? first + j.subs * C::W : j.np;
  f16x8 u[2][4];                                           // the block, on its way to LDS: 4 chunks of each plane
  auto fetch = [&](int j0) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) { const int id = k * C::NT + threadIdx.x; u[q][k] = *reinterpret_cast<const f16x8*>(w.x[q] + (int64_t)(id >> 4) * j.np + j0 + (id & 15) * 8); }
  };
  fetch(first);
  f32x4 acc[C::AR][C::AC] = {};
  const f32x4* from = reinterpret_cast<const f32x4*>(w.slab[gen]) + threadIdx.x;
#pragma unroll 4
  for (int q = 0; q < j.blocks; ++q)
#pragma unroll
    for (int i = 0; i < C::AR; ++i)
#pragma unroll
      for (int k = 0; k < C::AC; ++k) acc[i][k] += from[(int64_t)q * (M * M / 4) + (i * C::AC + k) * C::NT];
  thin_poly<C, M>(s, acc, cb, cc);
#pragma unroll
  for (int i = 0; i < C::AR; ++i)
#pragma unroll
    for (int k = 0; k < C::AC; ++k) acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int j0 = first; j0 < end; j0 += C::W) {
    if (j0 != first) { fetch(j0); __syncthreads(); }       // the block before has been read
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) { const int id = k * C::NT + threadIdx.x; *reinterpret_cast<f16x8*>(s.x[q] + (id >> 4) * C::PX + (id & 15) * 8) = u[q][k]; }
    __syncthreads();
    thin_update<C, M, LAST, T, MUON>(s, p, j, z, j0, ca);
    if (!LAST) {
      thin_keep<C, M>(s, w, j.np, j0);
      __syncthreads();
      thin_square<C, M, C::PX>(acc, s.x, C::W / 32);
    }
  }
  if (!LAST) thin_share<C>(acc, w.slab[gen ^ 1] + (int64_t)b * M * M);
}
