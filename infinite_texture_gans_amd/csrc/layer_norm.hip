// Layer norm over the channels of a row, forward and backward (gfx950).
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  r = 1 / sqrt(var + eps),  xh = (x - mean) r,  u = xh w + b,  y = act(u)
//   du = dy act'(u),  g = du w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum over rows of du xh,  db = sum over rows of du
//
// Statistics, sums and products are fp32 whatever the tensors' type; the variance is taken around the mean of the row (a second
// sweep over values that are already on the chip), never as a difference of moments.  Every sum has a fixed order: results do
// not change from call to call.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include "itg_common.h"

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

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }
template <> __device__ __forceinline__ float to_f<__hip_bfloat16>(__hip_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

__device__ __forceinline__ float act_slope_at(float u, int act, float slope) {
  if (act == ITG_ACT_LRELU) return u > 0.f ? 1.f : slope;
  if (act == ITG_ACT_TANH) { const float t = tanhf(u); return 1.f - t * t; }
  return 1.f;
}

// sum over the workgroup's 256 threads, the same value in every thread; `lds` holds 4 floats and may be re-used after the call
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// ---- any row length: one workgroup per row, the row is swept again from the cache for every quantity
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_fwd_any_kernel(LnP p) {
  __shared__ float lds[4];
  const T* X = (const T*)p.x;
  const W* w = (const W*)p.w; const W* b = (const W*)p.b;
  const float inv = 1.f / (float)p.c;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = X + row * p.ldx;
    float s = 0.f;
    for (int i = threadIdx.x; i < p.c; i += 256) s += to_f(x[i]);
    const float mean = block_sum(s, lds) * inv;
    s = 0.f;
    for (int i = threadIdx.x; i < p.c; i += 256) { const float d = to_f(x[i]) - mean; s = fmaf(d, d, s); }
    const float r = 1.f / sqrtf(block_sum(s, lds) * inv + p.eps);
    T* y = (T*)p.y + row * p.ldy;
    for (int i = threadIdx.x; i < p.c; i += 256) {
      const float u = fmaf((to_f(x[i]) - mean) * r, w ? to_f(w[i]) : 1.f, b ? to_f(b[i]) : 0.f);
      y[i] = from_f<T>(act_apply(u, p.act, p.slope));
    }
    for (int i = threadIdx.x; i < p.pad; i += 256) y[p.c + i] = from_f<T>(0.f);
    if (p.stat && threadIdx.x == 0) { p.stat[2 * row] = mean; p.stat[2 * row + 1] = r; }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_dx_any_kernel(LnP p) {
  __shared__ float lds[4];
  const W* w = (const W*)p.w; const W* b = (const W*)p.b;
  const float inv = 1.f / (float)p.c;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = (const T*)p.x + row * p.ldx;
    const T* dy = (const T*)p.dy + row * p.lddy;
    const float mean = p.stat[2 * row], r = p.stat[2 * row + 1];
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < p.c; i += 256) {
      const float xh = (to_f(x[i]) - mean) * r, wi = w ? to_f(w[i]) : 1.f;
      const float g = to_f(dy[i]) * act_slope_at(fmaf(xh, wi, b ? to_f(b[i]) : 0.f), p.act, p.slope) * wi;
      s1 += g; s2 = fmaf(g, xh, s2);
    }
    const float m1 = block_sum(s1, lds) * inv, m2 = block_sum(s2, lds) * inv;
    T* dx = (T*)p.y + row * p.ldy;
    for (int i = threadIdx.x; i < p.c; i += 256) {
      const float xh = (to_f(x[i]) - mean) * r, wi = w ? to_f(w[i]) : 1.f;
      const float g = to_f(dy[i]) * act_slope_at(fmaf(xh, wi, b ? to_f(b[i]) : 0.f), p.act, p.slope) * wi;
      dx[i] = from_f<T>(r * (g - m1 - xh * m2));
    }
    for (int i = threadIdx.x; i < p.pad; i += 256) dx[p.c + i] = from_f<T>(0.f);
  }
}

// shares of dw | db: a thread owns one channel and a chunk of the rows
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_dw_any_kernel(LnP p, int64_t chunk) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.c) return;
  const int64_t r0 = blockIdx.y * chunk, r1 = r0 + chunk < p.rows ? r0 + chunk : p.rows;
  const float wi = p.w ? to_f(((const W*)p.w)[i]) : 1.f, bi = p.b ? to_f(((const W*)p.b)[i]) : 0.f;
  float dw = 0.f, db = 0.f;
  for (int64_t row = r0; row < r1; ++row) {
    const float xh = (to_f(((const T*)p.x)[row * p.ldx + i]) - p.stat[2 * row]) * p.stat[2 * row + 1];
    const float du = to_f(((const T*)p.dy)[row * p.lddy + i]) * act_slope_at(fmaf(xh, wi, bi), p.act, p.slope);
    dw = fmaf(du, xh, dw); db += du;
  }
  float* part = p.part + (int64_t)blockIdx.y * 2 * p.c;
  part[i] = dw; part[p.c + i] = db;
}

// dw | db = the shares added in chunk order: 64 channels x 16 share lanes per workgroup
template <typename W>
__global__ __launch_bounds__(1024) void ln_dw_reduce_kernel(const float* __restrict__ part, int chunks, int c, W* dw, W* db, int acc) {
  __shared__ float lds[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), lane = threadIdx.x >> 6;
  float s = 0.f;
  if (col < 2 * c)
    for (int k = lane; k < chunks; k += 16) s += part[(int64_t)k * 2 * c + col];
  lds[lane][threadIdx.x & 63] = s;
  __syncthreads();
  if (lane == 0 && col < 2 * c) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += lds[k][threadIdx.x];
    W* out = col < c ? dw : db;
    const int i = col < c ? col : col - c;
    if (out) out[i] = from_f<W>(acc ? to_f(out[i]) + v : v);
  }
}

constexpr int LN_CHUNKS = 256;      // at most this many shares of dw | db
inline int ln_chunks(int64_t rows) { return (int)(rows < LN_CHUNKS ? rows : LN_CHUNKS); }
inline unsigned ln_grid(int64_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

template <typename T, typename W>
int ln_fwd_t(const LnP& p, hipStream_t s) {
  hipLaunchKernelGGL((ln_fwd_any_kernel<T, W>), dim3(ln_grid(p.rows)), dim3(256), 0, s, p);
  ITG_CHECK_LAUNCH();
  return ITG_OK;
}

template <typename T, typename W>
int ln_bwd_t(const LnP& p, void* dw, void* db, int acc, hipStream_t s) {
  if (p.y) {
    hipLaunchKernelGGL((ln_dx_any_kernel<T, W>), dim3(ln_grid(p.rows)), dim3(256), 0, s, p);
    ITG_CHECK_LAUNCH();
  }
  if (dw || db) {
    const int64_t chunk = (p.rows + ln_chunks(p.rows) - 1) / ln_chunks(p.rows);
    const int chunks = (int)((p.rows + chunk - 1) / chunk);
    hipLaunchKernelGGL((ln_dw_any_kernel<T, W>), dim3((p.c + 255) / 256, chunks), dim3(256), 0, s, p, chunk);
    ITG_CHECK_LAUNCH();
    hipLaunchKernelGGL((ln_dw_reduce_kernel<W>), dim3((2 * p.c + 63) / 64), dim3(1024), 0, s, p.part, chunks, p.c, (W*)dw, (W*)db, acc);
    ITG_CHECK_LAUNCH();
  }
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
    typedef __hip_bfloat16 T;                                                   \
    if (param_dtype == ITG_F32) { typedef float W; return CALL; }               \
    typedef __hip_bfloat16 W; return CALL;                                      \
  }                                                                             \
  typedef _Float16 T;                                                           \
  if (param_dtype == ITG_F32) { typedef float W; return CALL; }                 \
  typedef _Float16 W; return CALL;

extern "C" {

int itg_layer_norm_fwd(const void* x, int64_t ldx, const void* gamma, const void* beta, void* y, int64_t ldy, float* mean_rstd,
                       int64_t rows, int c, int pad, int dtype, int param_dtype, float eps, int act, float slope, void* stream) {
  int rc;
  if ((rc = ln_check(rows, c, 0, ldx, dtype, param_dtype, act)) || (rc = ln_check(rows, c, pad, ldy, dtype, param_dtype, act))) return rc;
  if (!x || !y || !(eps >= 0.f)) return ITG_ERR_ARG;
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
  return (int64_t)ln_chunks(rows) * 2 * c;
}

int itg_layer_norm_bwd(const void* x, int64_t ldx, const void* dy, int64_t lddy, const float* mean_rstd, const void* gamma,
                       const void* beta, void* dx, int64_t lddx, void* dgamma, void* dbeta, int accumulate, int64_t rows, int c,
                       int pad, int dtype, int param_dtype, int act, float slope, float* workspace, int64_t workspace_floats,
                       void* stream) {
  int rc;
  if ((rc = ln_check(rows, c, 0, ldx, dtype, param_dtype, act)) || (rc = ln_check(rows, c, 0, lddy, dtype, param_dtype, act)) ||
      (dx && (rc = ln_check(rows, c, pad, lddx, dtype, param_dtype, act)))) return rc;
  if (!x || !dy || !mean_rstd) return ITG_ERR_ARG;
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
