// Layer norm over the channels of a row, forward and backward (gfx950).
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  r = 1 / sqrt(var + eps),  xh = (x - mean) r,  u = xh w + b,  y = act(u)
//   du = dy act'(u),  g = du w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum over rows of du xh,  db = sum over rows of du
//
// Statistics, sums and products are fp32 whatever the tensors' type; the variance is taken around the mean of the row (a second
// sweep over values that are already on the chip), never as a difference of moments.  Every sum has a fixed order: results do
// not change from call to call.
#include "layer_norm_rows.h"

namespace {

struct LnP {
  const void* x; const void* dy; const void* w; const void* b;
  void* y;                    // forward: y, backward: dx (or NULL)
  float* stat;                // mean | rstd of every row: [rows][2]
  float* part;                // backward: [chunks][2][c] shares of dw | db
  int64_t rows, ldx, lddy, ldy;
  int c, pad;                 // pad: zero channels written behind c
  float eps, slope;
  int act;
};

__device__ __forceinline__ float act_slope_at(float u, int act, float slope) {
  if (act == ITG_ACT_LRELU) return u > 0.f ? 1.f : slope;
  if (act == ITG_ACT_TANH) { const float t = tanhf(u); return 1.f - t * t; }
  return 1.f;
}

// The R vectors of a thread in row `q`.  A thread that has none reads the row's last one, and ln_take makes zeros of it: a load behind
// a branch is waited for at the branch's end.
template <typename T, int V, int R>
__device__ __forceinline__ void ln_fetch(const T* q, const int (&off)[R], Held<T, V> (&u)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) u[r].load(q + off[r]);
}

template <typename T, int V, int R, bool MASK>
__device__ __forceinline__ void ln_take(const Held<T, V> (&u)[R], const int (&hi)[R], const Held<T, V> (&mine)[R], Held<T, V> (&k)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < Held<T, V>::N; ++i) k[r].w[i] = MASK ? u[r].w[i] & mine[r].w[i] : hi[r] > 0 ? u[r].w[i] : 0u;
}

// the bits of a vector's values in front of `hi`
template <typename T, int V>
__device__ __forceinline__ void ln_bits(int hi, Held<T, V>& m) {
#pragma unroll
  for (int i = 0; i < Held<T, V>::N; ++i) m.w[i] = 0u;
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (e < hi) m.w[e * sizeof(T) / 4] |= sizeof(T) == 4 ? ~0u : 0xffffu << (16 * (e & 1));
}

template <typename T, int V, bool MASK>
__device__ __forceinline__ void ln_store(T* q, const float (&f)[V], const Held<T, V>& mine) {
  Pack<T, V> u;
#pragma unroll
  for (int e = 0; e < V; ++e) u.v[e] = (T)f[e];
  if (MASK) {
    Held<T, V> k = {};
    __builtin_memcpy(&k, &u, sizeof(u));
#pragma unroll
    for (int i = 0; i < Held<T, V>::N; ++i) k.w[i] &= mine.w[i];
    __builtin_memcpy(&u, &k, sizeof(u));
  }
  *reinterpret_cast<Pack<T, V>*>(q) = u;
}

// V values of gamma or beta, `none` without one.  A vector of a padded row that ends in the padding (hi < V) is read value by value.
template <typename W, int V, bool ANY>
__device__ __forceinline__ void ln_param(const void* q, int off, int hi, float none, float (&f)[V]) {
  Pack<W, V> u = {};
  const W* at = (const W*)q + off;
  if (q && hi > 0) {
    if (!ANY || hi == V) {
      u = *reinterpret_cast<const Pack<W, V>*>(at);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < hi) u.v[e] = at[e];
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = q ? (float)u.v[e] : none;
}

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}

// sum over aligned groups of G <= 64 lanes, in every lane: cross-lane moves inside 16 lanes, two shuffles beyond
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if (G >= 2) v += dpp<0xB1>(v);        // lane ^ 1
  if (G >= 4) v += dpp<0x4E>(v);        // lane ^ 2
  if (G >= 8) v += dpp<0x141>(v);       // mirror in 8: the other four
  if (G >= 16) v += dpp<0x140>(v);      // mirror in 16: the other eight
  if (G >= 32) v += __shfl_xor(v, 16, 64);
  if (G >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// sum over the TPR threads of a row.  TPR > 64: through LDS, `red` = this call's TPR / 64 floats, one barrier
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = group_sum<(TPR < 64 ? TPR : 64)>(v);
  if (TPR <= 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < (TPR > 64 ? TPR / 64 : 1); ++k) s += red[k];
  return s;
}

// two sums at once, `red` = 2 TPR / 64 floats, one barrier
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
  a = group_sum<(TPR < 64 ? TPR : 64)>(a);
  b = group_sum<(TPR < 64 ? TPR : 64)>(b);
  if (TPR <= 64) return;
  if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = a; red[TPR / 64 + (threadIdx.x >> 6)] = b; }
  __syncthreads();
  a = b = 0.f;
#pragma unroll
  for (int k = 0; k < (TPR > 64 ? TPR / 64 : 1); ++k) { a += red[k]; b += red[TPR / 64 + k]; }
}

// a thread's row among those of its workgroup; from a wave per row on the same in every lane, and known to be: addresses then are a
// scalar base and 32 bits a lane
template <int TPR> __device__ __forceinline__ int ln_group() {
  return TPR > 64 ? 0 : TPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x / TPR;
}

// What a row needs beyond its values: nothing, masks (V does not divide it), or an activation too.  Each is a kernel of its own: at 2
// bytes a value instructions are time (forward, bf16: 16384 x 4096 takes 43.0 us plain, 49.3 with the activation, 53.6 where masks and
// the activation's kind are looked at for every value; 60000 x 333 19.7 us where a mask is a factor and an AND, 25.7 where it is two
// comparisons a value).
enum { LN_PLAIN = 0, LN_MASK = 1, LN_ACT = 2 };

template <typename T, typename W, int V, int TPR, int R, int KIND>
__global__ __launch_bounds__(TPR > 64 ? TPR : 256) void ln_fwd_kernel(LnP p) {
  constexpr int NT = TPR > 64 ? TPR : 256, GROUPS = NT / TPR;
  __shared__ float red[4][TPR > 64 ? TPR / 64 : 1];      // two sums per row, two rows' worth: a row's sums outlive the next row's first barrier
  const LnV lv = ln_vectors(p.c, p.pad, V);
  const int tid = TPR > 64 ? threadIdx.x : threadIdx.x % TPR;
  constexpr bool MASK = KIND != LN_PLAIN;
  int off[R], lo[R], hi[R];
  float w[R][V], b[R][V], m[R][V];      // m: 1 for the values a thread counts, 0 for those it shares with a neighbour and padding
  Held<T, V> mine[R];                   // the bits of the values it reads and writes
#pragma unroll
  for (int r = 0; r < R; ++r) {
    ln_place(lv, tid + r * TPR, V, off[r], lo[r], hi[r]);
    if (MASK) {
      ln_bits<T, V>(hi[r], mine[r]);
#pragma unroll
      for (int e = 0; e < V; ++e) m[r][e] = e >= lo[r] && e < hi[r] ? 1.f : 0.f;
    }
  }
  const float inv = 1.f / (float)p.c;
  int flip = 0;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + ln_group<TPR>();
  Held<T, V> u[R] = {};
  if (row < p.rows) ln_fetch<T, V, R>((const T*)p.x + row * p.ldx, off, u);
#pragma unroll
  for (int r = 0; r < R; ++r) { ln_param<W, V, MASK>(p.w, off[r], hi[r], 1.f, w[r]); ln_param<W, V, MASK>(p.b, off[r], hi[r], 0.f, b[r]); }
  const float below = p.act == ITG_ACT_LRELU ? p.slope : 1.f;
  for (; row < p.rows; row += step, flip ^= 2) {
    float f[R][V], s = 0.f;
    Held<T, V> k[R];
    ln_take<T, V, R, MASK>(u, hi, mine, k);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[r][e] = k[r].at(e);
        s = MASK ? fmaf(f[r][e], m[r][e], s) : s + f[r][e];      // a vector past the row's end holds zeros
      }
    // the next row is on its way while this one is reduced and written
    if (row + step < p.rows) ln_fetch<T, V, R>((const T*)p.x + (row + step) * p.ldx, off, u);
    const float mean = row_sum<TPR>(s, red[flip]) * inv;
    s = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float q = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[r][e] -= mean;
        q = fmaf(MASK ? f[r][e] * m[r][e] : f[r][e], f[r][e], q);
      }
      s += MASK || hi[r] > 0 ? q : 0.f;
    }
    const float rs = 1.f / sqrtf(row_sum<TPR>(s, red[flip + 1]) * inv + p.eps);
    T* y = (T*)p.y + row * p.ldy;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (hi[r] <= 0) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[r][e] = fmaf(f[r][e] * rs, w[r][e], b[r][e]);
        if (KIND == LN_ACT) f[r][e] = f[r][e] > 0.f ? f[r][e] : f[r][e] * below;
      }
      if (KIND == LN_ACT && p.act == ITG_ACT_TANH) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[r][e] = tanhf(f[r][e]);
      }
      ln_store<T, V, MASK>(y + off[r], f[r], mine[r]);
    }
    if (MASK && p.pad && lv.hi_last == V)
      for (int i = tid; i < p.pad; i += TPR) y[p.c + i] = (T)0.f;
    if (p.stat && tid == 0) { p.stat[2 * row] = mean; p.stat[2 * row + 1] = rs; }
  }
}

// dx, and this workgroup's share of dw | db (`part`), which a thread sums over the rows it sees for the channels it holds.
// At 16 channels in each of 1024 threads (rows of 8193 .. 16384 16-bit values) the row stays in its own 16 bits between the two
// sweeps and gamma in its own type, and the next row is fetched behind the last sweep: fp32 copies and a row under way do not fit
// the 128 registers that 1024 threads have.  Nor does this quite: 4 to 12 registers spill without masks, 14 to 47 with masks or an
// activation (20 to 164 bytes of scratch a thread), some of them reloaded in the row loop (4096 x 12288 bf16: 88 us against 62 of the
// bytes alone; swept three times by the kernels for any length 142).
template <typename T, typename W, int V, int TPR, int R, int KIND>
__global__ __launch_bounds__(TPR > 64 ? TPR : 256) void ln_bwd_kernel(LnP p) {
  constexpr int NT = TPR > 64 ? TPR : 256, GROUPS = NT / TPR;
  constexpr bool TIGHT = R * V >= 16 && TPR == 1024, MASK = KIND != LN_PLAIN, ACT = KIND == LN_ACT;
  __shared__ float red[4][TPR > 64 ? TPR / 64 : 1];
  const LnV lv = ln_vectors(p.c, p.pad, V);
  const int tid = TPR > 64 ? threadIdx.x : threadIdx.x % TPR;
  int off[R], lo[R], hi[R];
  float w[R][V], b[R][V], aw[R][V], ab[R][V], m[R][V];
  Held<T, V> mine[R];
  Held<W, V> tw[R] = {}, tb[R] = {};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    ln_place(lv, tid + r * TPR, V, off[r], lo[r], hi[r]);
    if (MASK) {
      ln_bits<T, V>(hi[r], mine[r]);
#pragma unroll
      for (int e = 0; e < V; ++e) m[r][e] = e >= lo[r] && e < hi[r] ? 1.f : 0.f;
    }
    if (TIGHT) {
      // (gamma and beta hold c values: a padded row's last vector ends behind them)
      if (hi[r] > 0 && p.w) tw[r].load_first((const W*)p.w + off[r], MASK ? hi[r] : V);
      if (ACT && hi[r] > 0 && p.b) tb[r].load_first((const W*)p.b + off[r], hi[r]);
    } else {
      ln_param<W, V, MASK>(p.w, off[r], hi[r], 1.f, w[r]);
      ln_param<W, V, MASK>(ACT ? p.b : nullptr, off[r], hi[r], 0.f, b[r]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) aw[r][e] = ab[r][e] = 0.f;
  }
  const float inv = 1.f / (float)p.c;
  int flip = 0;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + ln_group<TPR>();
  Held<T, V> ux[R] = {}, ug[R] = {};
  float mean = 0.f, rs = 0.f;
  auto fetch = [&](int64_t at) {
    ln_fetch<T, V, R>((const T*)p.x + at * p.ldx, off, ux);
    ln_fetch<T, V, R>((const T*)p.dy + at * p.lddy, off, ug);
    mean = p.stat[2 * at]; rs = p.stat[2 * at + 1];
  };
  auto gain = [&](int r, int e) { return TIGHT ? p.w ? tw[r].at(e) : 1.f : w[r][e]; };
  // xh, and the gradient in front of the activation
  auto at_u = [&](int r, int e, const Held<T, V>& px, const Held<T, V>& pg, float m, float s, float& xh, float& du) {
    xh = (px.at(e) - m) * s;
    du = pg.at(e);
    if (ACT) {
      const float u = fmaf(xh, gain(r, e), TIGHT ? tb[r].at(e) : b[r][e]);
      if (p.act == ITG_ACT_TANH) { const float t = tanhf(u); du *= 1.f - t * t; }
      else du *= u > 0.f ? 1.f : p.slope;
    }
  };
  if (row < p.rows) fetch(row);
  for (; row < p.rows; row += step, flip ^= 2) {
    float xh[R][V], g[R][V], s1 = 0.f, s2 = 0.f;
    const float r_now = rs, m_now = mean;
    Held<T, V> kx[R], kg[R];
    ln_take<T, V, R, MASK>(ux, hi, mine, kx);
    ln_take<T, V, R, MASK>(ug, hi, mine, kg);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (TIGHT) { kx[r].renew(); kg[r].renew(); tw[r].renew(); if (ACT) tb[r].renew(); }
#pragma unroll
      for (int e = 0; e < V; ++e) {      // a vector past the row's end holds zeros in dy
        float h, du;
        at_u(r, e, kx[r], kg[r], m_now, r_now, h, du);
        xh[r][e] = h;
        aw[r][e] = fmaf(du, h, aw[r][e]);      // (of a value that a neighbour counts, too: left out at the end)
        ab[r][e] += du;
        g[r][e] = du * gain(r, e);
        const float gi = !MASK ? g[r][e] : TIGHT ? (e >= lo[r] && e < hi[r] ? g[r][e] : 0.f) : g[r][e] * m[r][e];
        s1 += gi;
        s2 = fmaf(gi, h, s2);
      }
    }
    if (TIGHT) {
#pragma unroll
      for (int r = 0; r < R; ++r) { kx[r].renew(); kg[r].renew(); tw[r].renew(); if (ACT) tb[r].renew(); }
    }
    // the next row is on its way while this one is reduced and written
    if (!TIGHT && row + step < p.rows) fetch(row + step);
    if (p.y) {
      if (TIGHT) { s1 = row_sum<TPR>(s1, red[flip]); s2 = row_sum<TPR>(s2, red[flip + 1]); }      // (both at once spill more)
      else row_sum2<TPR>(s1, s2, red[flip]);
      const float m1 = s1 * inv, m2 = s2 * inv;
      T* dx = (T*)p.y + row * p.ldy;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (hi[r] <= 0) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (TIGHT) { at_u(r, e, kx[r], kg[r], m_now, r_now, xh[r][e], g[r][e]); g[r][e] *= gain(r, e); }
          g[r][e] = r_now * (g[r][e] - m1 - xh[r][e] * m2);
        }
        ln_store<T, V, MASK>(dx + off[r], g[r], mine[r]);
      }
      if (MASK && p.pad && lv.hi_last == V)
        for (int i = tid; i < p.pad; i += TPR) dx[p.c + i] = (T)0.f;
    }
    if (TIGHT && row + step < p.rows) fetch(row + step);
  }
  if (!p.part) return;
  // the row groups of this workgroup: lanes of a wave by shuffles, waves in order through LDS
  float* part = p.part + (int64_t)blockIdx.x * 2 * p.c;
  constexpr int WAVES = TPR <= 64 ? NT / 64 : 1;
  __shared__ float acc[WAVES > 1 ? WAVES - 1 : 1][2][WAVES > 1 ? (TPR < 64 ? TPR : 64) * R * V : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (TPR < 64) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < V; ++e)
#pragma unroll
        for (int o = TPR; o < 64; o <<= 1) { aw[r][e] += __shfl_xor(aw[r][e], o, 64); ab[r][e] += __shfl_xor(ab[r][e], o, 64); }
  }
  if (WAVES > 1) {
    if (wave > 0 && lane < TPR) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) { acc[wave - 1][0][(r * V + e) * (TPR < 64 ? TPR : 64) + tid] = aw[r][e]; acc[wave - 1][1][(r * V + e) * (TPR < 64 ? TPR : 64) + tid] = ab[r][e]; }
    }
    __syncthreads();
    if (wave > 0 || lane >= TPR) return;
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float vw = aw[r][e], vb = ab[r][e];
      if (WAVES > 1) {
#pragma unroll
        for (int k = 0; k < WAVES - 1; ++k) { vw += acc[k][0][(r * V + e) * (TPR < 64 ? TPR : 64) + tid]; vb += acc[k][1][(r * V + e) * (TPR < 64 ? TPR : 64) + tid]; }
      }
      if (e >= lo[r] && e < hi[r]) { part[off[r] + e] = vw; part[p.c + off[r] + e] = vb; }
    }
}

// ---- any row length: one workgroup of 1024 threads per row, which sweeps the row again (from the cache) for every quantity
constexpr int LN_ANY = 1024;

template <int N> struct Width { static constexpr int value = N; };

// f(first channel, Width) over the row's whole vectors of V values, then over the values behind them
template <int V, typename F>
__device__ __forceinline__ void ln_sweep(int c, F f) {
  const int full = c / V;
  for (int i = threadIdx.x; i < full; i += LN_ANY) f(i * V, Width<V>{});
  for (int i = full * V + threadIdx.x; i < c; i += LN_ANY) f(i, Width<1>{});
}

template <typename T, int N> __device__ __forceinline__ Pack<T, N> ln_at(const T* q) { return *reinterpret_cast<const Pack<T, N>*>(q); }

template <typename T, typename W, int V>
__global__ __launch_bounds__(LN_ANY) void ln_fwd_any_kernel(LnP p) {
  __shared__ float red[4][LN_ANY / 64];
  const W* w = (const W*)p.w; const W* b = (const W*)p.b;
  const float inv = 1.f / (float)p.c;
  int flip = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, flip ^= 2) {
    const T* x = (const T*)p.x + row * p.ldx;
    float s = 0.f;
    ln_sweep<V>(p.c, [&](int at, auto width) {
      constexpr int N = decltype(width)::value;
      const auto u = ln_at<T, N>(x + at);
#pragma unroll
      for (int e = 0; e < N; ++e) s += (float)u.v[e];
    });
    const float mean = row_sum<LN_ANY>(s, red[flip]) * inv;
    s = 0.f;
    ln_sweep<V>(p.c, [&](int at, auto width) {
      constexpr int N = decltype(width)::value;
      const auto u = ln_at<T, N>(x + at);
#pragma unroll
      for (int e = 0; e < N; ++e) { const float d = (float)u.v[e] - mean; s = fmaf(d, d, s); }
    });
    const float r = 1.f / sqrtf(row_sum<LN_ANY>(s, red[flip + 1]) * inv + p.eps);
    T* y = (T*)p.y + row * p.ldy;
    ln_sweep<V>(p.c, [&](int at, auto width) {
      constexpr int N = decltype(width)::value;
      auto u = ln_at<T, N>(x + at);
      Pack<W, N> uw, ub;
      if (w) uw = ln_at<W, N>(w + at);
      if (b) ub = ln_at<W, N>(b + at);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = fmaf(((float)u.v[e] - mean) * r, w ? (float)uw.v[e] : 1.f, b ? (float)ub.v[e] : 0.f);
        u.v[e] = (T)act_apply(v, p.act, p.slope);
      }
      *reinterpret_cast<Pack<T, N>*>(y + at) = u;
    });
    for (int i = threadIdx.x; i < p.pad; i += LN_ANY) y[p.c + i] = (T)0.f;
    if (p.stat && threadIdx.x == 0) { p.stat[2 * row] = mean; p.stat[2 * row + 1] = r; }
  }
}

template <typename T, typename W, int V>
__global__ __launch_bounds__(LN_ANY) void ln_dx_any_kernel(LnP p) {
  __shared__ float red[4][LN_ANY / 64];
  const W* w = (const W*)p.w; const W* b = (const W*)p.b;
  const float inv = 1.f / (float)p.c;
  int flip = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, flip ^= 2) {
    const T* x = (const T*)p.x + row * p.ldx;
    const T* dy = (const T*)p.dy + row * p.lddy;
    const float mean = p.stat[2 * row], r = p.stat[2 * row + 1];
    float s1 = 0.f, s2 = 0.f;
    ln_sweep<V>(p.c, [&](int at, auto width) {
      constexpr int N = decltype(width)::value;
      const auto ux = ln_at<T, N>(x + at), ug = ln_at<T, N>(dy + at);
      Pack<W, N> uw, ub;
      if (w) uw = ln_at<W, N>(w + at);
      if (b && p.act) ub = ln_at<W, N>(b + at);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float xh = ((float)ux.v[e] - mean) * r, wi = w ? (float)uw.v[e] : 1.f;
        float g = (float)ug.v[e] * wi;
        if (p.act) g *= act_slope_at(fmaf(xh, wi, b ? (float)ub.v[e] : 0.f), p.act, p.slope);
        s1 += g; s2 = fmaf(g, xh, s2);
      }
    });
    row_sum2<LN_ANY>(s1, s2, red[flip]);
    const float m1 = s1 * inv, m2 = s2 * inv;
    T* dx = (T*)p.y + row * p.ldy;
    ln_sweep<V>(p.c, [&](int at, auto width) {
      constexpr int N = decltype(width)::value;
      auto ux = ln_at<T, N>(x + at);
      const auto ug = ln_at<T, N>(dy + at);
      Pack<W, N> uw, ub;
      if (w) uw = ln_at<W, N>(w + at);
      if (b && p.act) ub = ln_at<W, N>(b + at);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float xh = ((float)ux.v[e] - mean) * r, wi = w ? (float)uw.v[e] : 1.f;
        float g = (float)ug.v[e] * wi;
        if (p.act) g *= act_slope_at(fmaf(xh, wi, b ? (float)ub.v[e] : 0.f), p.act, p.slope);
        ux.v[e] = (T)(r * (g - m1 - xh * m2));
      }
      *reinterpret_cast<Pack<T, N>*>(dx + at) = ux;
    });
    for (int i = threadIdx.x; i < p.pad; i += LN_ANY) dx[p.c + i] = (T)0.f;
  }
}

// shares of dw | db: a thread owns N channels (the last one starts at c - N and leaves what its neighbour holds) and a chunk of the rows
template <typename T, typename W, int N>
__global__ __launch_bounds__(256) void ln_dw_any_kernel(LnP p, int64_t chunk) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i * N >= p.c) return;
  const int at = i * N + N <= p.c ? i * N : p.c - N, lo = i * N - at;
  const int64_t r0 = blockIdx.y * chunk, r1 = r0 + chunk < p.rows ? r0 + chunk : p.rows;
  float w[N], b[N], dw[N], db[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    w[e] = p.w ? (float)((const W*)p.w)[at + e] : 1.f;
    b[e] = p.b ? (float)((const W*)p.b)[at + e] : 0.f;
    dw[e] = db[e] = 0.f;
  }
#pragma unroll 2
  for (int64_t row = r0; row < r1; ++row) {
    const auto ux = ln_at<T, N>((const T*)p.x + row * p.ldx + at), ug = ln_at<T, N>((const T*)p.dy + row * p.lddy + at);
    const float mean = p.stat[2 * row], r = p.stat[2 * row + 1];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float xh = ((float)ux.v[e] - mean) * r;
      float du = (float)ug.v[e];
      if (p.act) du *= act_slope_at(fmaf(xh, w[e], b[e]), p.act, p.slope);
      dw[e] = fmaf(du, xh, dw[e]); db[e] += du;
    }
  }
  float* part = p.part + (int64_t)blockIdx.y * 2 * p.c;
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e >= lo) { part[at + e] = dw[e]; part[p.c + at + e] = db[e]; }
}

// dw | db = the shares added in a fixed order: 16 channels x 64 share lanes per workgroup
template <typename W>
__global__ __launch_bounds__(1024) void ln_dw_reduce_kernel(const float* __restrict__ part, int chunks, int c, W* dw, W* db, int acc) {
  __shared__ float lds[64][17];
  const int k = threadIdx.x & 15, col = blockIdx.x * 16 + k, lane = threadIdx.x >> 4;
  float s = 0.f;
  if (col < 2 * c) {
#pragma unroll 4
    for (int q = lane; q < chunks; q += 64) s += part[(int64_t)q * 2 * c + col];
  }
  lds[lane][k] = s;
  __syncthreads();
  if (lane < 16) {                                 // 16 lanes x 4 shares, then the 16 sums of a channel (lanes of one row of 16)
    const int ch = lane;                           // transposed: thread (lane, k) takes channel `lane`, shares k, k + 16, ...
    float v = (lds[k][ch] + lds[k + 16][ch]) + (lds[k + 32][ch] + lds[k + 48][ch]);
    v = group_sum<16>(v);
    const int out_col = blockIdx.x * 16 + ch;
    if (k == 0 && out_col < 2 * c) {
      W* out = out_col < c ? dw : db;
      const int i = out_col < c ? out_col : out_col - c;
      if (out) out[i] = (W)(acc ? (float)out[i] + v : v);
    }
  }
}

inline unsigned ln_grid(int64_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

template <int V> inline int ln_kind(const LnP& p) { return p.act != ITG_ACT_NONE ? LN_ACT : p.c % V != 0 || p.pad != 0 ? LN_MASK : LN_PLAIN; }

template <typename T, typename W, int V, int TPR, int R>
int ln_fwd_run(const LnP& p, hipStream_t s) {
  constexpr int NT = TPR > 64 ? TPR : 256, GROUPS = NT / TPR;
  const int64_t need = (p.rows + GROUPS - 1) / GROUPS, most = 256 * (2048 / NT);
  const dim3 grid((unsigned)(need < most ? need : most));
  const int kind = ln_kind<V>(p);
  if (kind == LN_ACT) hipLaunchKernelGGL((ln_fwd_kernel<T, W, V, TPR, R, LN_ACT>), grid, dim3(NT), 0, s, p);
  else if (kind == LN_MASK) hipLaunchKernelGGL((ln_fwd_kernel<T, W, V, TPR, R, LN_MASK>), grid, dim3(NT), 0, s, p);
  else hipLaunchKernelGGL((ln_fwd_kernel<T, W, V, TPR, R, LN_PLAIN>), grid, dim3(NT), 0, s, p);
  ITG_CHECK_LAUNCH();
  return ITG_OK;
}

// Threads per row and vectors per thread: as few threads as hold the row at one vector each up to a wave; beyond, workgroups of
// 128 .. 1024 threads at two vectors each.  The backward pass's: ln_bwd_threads.
template <typename T, typename W>
int ln_fwd_t(const LnP& p, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (p.c < V && !ln_padded(p.c, p.pad, V)) return p.c <= 4 ? ln_fwd_run<T, W, 1, 4, 1>(p, s) : ln_fwd_run<T, W, 1, 8, 1>(p, s);
  const int nv = (p.c + V - 1) / V;
  if (nv <= 4) return ln_fwd_run<T, W, V, 4, 1>(p, s);
  if (nv <= 8) return ln_fwd_run<T, W, V, 8, 1>(p, s);
  if (nv <= 16) return ln_fwd_run<T, W, V, 16, 1>(p, s);
  if (nv <= 32) return ln_fwd_run<T, W, V, 32, 1>(p, s);
  if (nv <= 64) return ln_fwd_run<T, W, V, 64, 1>(p, s);
  if (nv <= 128) return ln_fwd_run<T, W, V, 64, 2>(p, s);
  if (nv <= 256) return ln_fwd_run<T, W, V, 128, 2>(p, s);
  if (nv <= 512) return ln_fwd_run<T, W, V, 256, 2>(p, s);
  if (nv <= 1024) return ln_fwd_run<T, W, V, 512, 2>(p, s);
  if (nv <= 2048) return ln_fwd_run<T, W, V, 1024, 2>(p, s);
  hipLaunchKernelGGL((ln_fwd_any_kernel<T, W, V>), dim3(ln_grid(p.rows)), dim3(LN_ANY), 0, s, p);
  ITG_CHECK_LAUNCH();
  return ITG_OK;
}

// rows in registers; a workgroup leaves one share of dw | db
template <typename T, typename W, int V, int TPR, int R>
int ln_bwd_run(const LnP& p, hipStream_t s) {
  constexpr int NT = TPR > 64 ? TPR : 256;
  const dim3 grid((unsigned)ln_bwd_groups(p.rows, TPR));
  const int kind = ln_kind<V>(p);
  if (kind == LN_ACT) hipLaunchKernelGGL((ln_bwd_kernel<T, W, V, TPR, R, LN_ACT>), grid, dim3(NT), 0, s, p);
  else if (kind == LN_MASK) hipLaunchKernelGGL((ln_bwd_kernel<T, W, V, TPR, R, LN_MASK>), grid, dim3(NT), 0, s, p);
  else hipLaunchKernelGGL((ln_bwd_kernel<T, W, V, TPR, R, LN_PLAIN>), grid, dim3(NT), 0, s, p);
  ITG_CHECK_LAUNCH();
  return ITG_OK;
}

template <typename T, typename W>
int ln_bwd_t(LnP p, void* dw, void* db, int acc, hipStream_t s) {
  constexpr int V = 16 / sizeof(T), K = V == 8 ? 1 : 2;      // K: vectors per thread of the workgroup sizes
  const int nv = (p.c + V - 1) / V, threads = ln_bwd_threads(p.rows, p.c, p.pad, V), chunks = ln_bwd_shares(p.rows, p.c, p.pad, V);
  const bool shares = dw || db;
  int rc = ITG_OK;
  if (!shares) p.part = nullptr;
  if (p.c < V && !ln_padded(p.c, p.pad, V)) rc = threads == 4 ? ln_bwd_run<T, W, 1, 4, 1>(p, s) : ln_bwd_run<T, W, 1, 8, 1>(p, s);
  else if (threads == 4) rc = ln_bwd_run<T, W, V, 4, 1>(p, s);
  else if (threads == 8) rc = ln_bwd_run<T, W, V, 8, 1>(p, s);
  else if (threads == 16) rc = ln_bwd_run<T, W, V, 16, 1>(p, s);
  else if (threads == 32) rc = ln_bwd_run<T, W, V, 32, 1>(p, s);
  else if (threads == 64) rc = nv <= 64 ? ln_bwd_run<T, W, V, 64, 1>(p, s) : ln_bwd_run<T, W, V, 64, 2>(p, s);
  else if (K == 2 && threads == 128) rc = ln_bwd_run<T, W, V, K == 2 ? 128 : 256, K>(p, s);
  else if (threads == 256) rc = ln_bwd_run<T, W, V, 256, K>(p, s);
  else if (threads == 512) rc = ln_bwd_run<T, W, V, 512, K>(p, s);
  else if (threads == 1024) rc = nv <= 1024 * K ? ln_bwd_run<T, W, V, 1024, K>(p, s) : ln_bwd_run<T, W, V, 1024, 2>(p, s);
  else {
    // (the shares read every row of dy and x, and dx may be written over either)
    if (shares) {
      hipLaunchKernelGGL((ln_dw_any_kernel<T, W, V>), dim3((nv + 255) / 256, chunks), dim3(256), 0, s, p, ln_bwd_chunk(p.rows, p.c, V));
      ITG_CHECK_LAUNCH();
    }
    if (p.y) {
      hipLaunchKernelGGL((ln_dx_any_kernel<T, W, V>), dim3(ln_grid(p.rows)), dim3(LN_ANY), 0, s, p);
      ITG_CHECK_LAUNCH();
    }
  }
  if (rc || !shares) return rc;
  hipLaunchKernelGGL((ln_dw_reduce_kernel<W>), dim3((2 * p.c + 15) / 16), dim3(1024), 0, s, p.part, chunks, p.c, (W*)dw, (W*)db, acc);
  ITG_CHECK_LAUNCH();
  return ITG_OK;
}

inline int ln_check(int64_t rows, int c, int pad, int64_t ld, int dtype, int pdtype, int act) {
  if (rows <= 0 || c <= 0 || pad < 0 || c > ITG_LN_MAX_C || pad > ITG_LN_MAX_C) return ITG_ERR_ARG;
  if (rows > 1 && ld < (int64_t)c + pad) return ITG_ERR_ARG;
  if (rows > ((int64_t)1 << 40) || ld > ((int64_t)1 << 40) || (rows > 1 && ld > (((int64_t)1 << 60) / rows))) return ITG_ERR_ARG;
  if (dtype < ITG_F32 || dtype > ITG_F16 || (pdtype != ITG_F32 && pdtype != dtype)) return ITG_ERR_ARG;
  if (act < ITG_ACT_NONE || act > ITG_ACT_TANH) return ITG_ERR_ARG;
  return ITG_OK;
}

inline bool misaligned(const void* q, int dtype) { return ((uintptr_t)q & (dtype == ITG_F32 ? 3 : 1)) != 0; }

}  // namespace

#define LN_TYPES(CALL)                                                          \
  if (dtype == ITG_F32) { typedef float T; typedef float W; return CALL; }      \
  if (dtype == ITG_BF16) {                                                      \
    typedef __bf16 T;                                                   \
    if (param_dtype == ITG_F32) { typedef float W; return CALL; }               \
    typedef __bf16 W; return CALL;                                      \
  }                                                                             \
  typedef _Float16 T;                                                           \
  if (param_dtype == ITG_F32) { typedef float W; return CALL; }                 \
  typedef _Float16 W; return CALL;

extern "C" {

int itg_layer_norm_fwd(const void* x, int64_t ldx, const void* gamma, const void* beta, void* y, int64_t ldy, float* mean_rstd,
                       int64_t rows, int c, int pad, int dtype, int param_dtype, float eps, int act, float slope, void* stream) {
  int rc;
  if ((rc = ln_check(rows, c, pad, ldx, dtype, param_dtype, act)) || (rc = ln_check(rows, c, pad, ldy, dtype, param_dtype, act))) return rc;
  if (!x || !y || !(eps >= 0.f) || (rows > 1 && y == x && ldy != ldx)) return ITG_ERR_ARG;
  if (misaligned(x, dtype) || misaligned(y, dtype) || misaligned(gamma, param_dtype) || misaligned(beta, param_dtype) ||
      misaligned(mean_rstd, ITG_F32)) return ITG_ERR_ALIGN;
  LnP p{};
  p.x = x; p.w = gamma; p.b = beta; p.y = y; p.stat = mean_rstd; p.rows = rows; p.ldx = ldx; p.ldy = ldy; p.c = c; p.pad = pad;
  p.eps = eps; p.act = act; p.slope = slope;
  hipStream_t s = (hipStream_t)stream;
  LN_TYPES((ln_fwd_t<T, W>(p, s)))
}

int64_t itg_layer_norm_bwd_workspace(int64_t rows, int c) {
  if (rows <= 0 || c <= 0 || c > ITG_LN_MAX_C) return ITG_ERR_ARG;
  return (int64_t)ln_bwd_most_shares(rows, c) * 2 * c;
}

int itg_layer_norm_bwd(const void* x, int64_t ldx, const void* dy, int64_t lddy, const float* mean_rstd, const void* gamma,
                       const void* beta, void* dx, int64_t lddx, void* dgamma, void* dbeta, int accumulate, int64_t rows, int c,
                       int pad, int dtype, int param_dtype, int act, float slope, float* workspace, int64_t workspace_floats,
                       void* stream) {
  int rc;
  if ((rc = ln_check(rows, c, pad, ldx, dtype, param_dtype, act)) || (rc = ln_check(rows, c, pad, lddy, dtype, param_dtype, act)) ||
      (dx && (rc = ln_check(rows, c, pad, lddx, dtype, param_dtype, act)))) return rc;
  if (!x || !dy || !mean_rstd) return ITG_ERR_ARG;
  if (rows > 1 && ((dx == x && lddx != ldx) || (dx == dy && lddx != lddy))) return ITG_ERR_ARG;
  if (misaligned(x, dtype) || misaligned(dy, dtype) || misaligned(dx, dtype) || misaligned(gamma, param_dtype) ||
      misaligned(beta, param_dtype) || misaligned(dgamma, param_dtype) || misaligned(dbeta, param_dtype) ||
      misaligned(mean_rstd, ITG_F32) || misaligned(workspace, ITG_F32)) return ITG_ERR_ALIGN;
  if ((dgamma || dbeta) && (!workspace || workspace_floats < itg_layer_norm_bwd_workspace(rows, c))) return ITG_ERR_WORKSPACE;
  if (!dx && !dgamma && !dbeta) return ITG_OK;
  LnP p{};
  p.x = x; p.dy = dy; p.w = gamma; p.b = beta; p.y = dx; p.stat = const_cast<float*>(mean_rstd); p.part = workspace; p.rows = rows;
  p.ldx = ldx; p.lddy = lddy; p.ldy = lddx; p.c = c; p.pad = pad; p.act = act; p.slope = slope;
  hipStream_t s = (hipStream_t)stream;
  LN_TYPES((ln_bwd_t<T, W>(p, dgamma, dbeta, accumulate, s)))
}

}  // extern "C"
