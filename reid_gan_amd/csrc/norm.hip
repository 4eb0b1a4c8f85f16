// Layer norm over the last axis, forward and backward (the token counterpart of the BatchNorm kernels).
//   forward   mu = mean x, r = 1 / sqrt(mean (x - mu)^2 + eps), xh = (x - mu) r, y = xh w + b
//   backward  dxh = dy w, dx = r (dxh - mean dxh - xh mean(dxh xh)), dw = sum_rows dy xh, db = sum_rows dy
// HBM-bound: forward reads and writes each element once, backward reads x and dy and writes dx once.  A row stays in
// registers between the statistics and the result (16-byte chunks, NV per lane); the variance is the mean of centred
// squares, so a large mean costs no precision.  The weight's gradient is summed where the row already is: every lane
// keeps the sums of its own columns over all rows its block takes, the block adds its row groups in LDS, and a second
// kernel adds the blocks' partial rows.  No atomics: the order of every sum is fixed.
//
// A row of up to 1024 elements in 16 bits is one wave's (two chunks a lane), so its statistics need no barrier; narrower rows
// share a wave, wider ones take 4 or 16.  Measured, 16384 rows of 1024 in bf16: forward 18.6 us (67 MB, 3.6 TB/s), backward
// 22.4 us (101 MB, 4.5 TB/s) + 4.0 us for the parameter gradients' partial rows (1024 of them; 512 were 26.4 + 4.7).  4099
// rows of 777 in fp32: 9.5, and 10.2 + 3.6 us.  16 rows of 512: 2.7 us.  (A forward kernel whose blocks
// walk several rows, the next row and the weights asked for early, took 18.9 us.)
#include "tokens.h"

// A group of LPR lanes (up to 64), or of WPR whole waves, owns a row.
template <int LPR, int WPR>
__device__ __forceinline__ float group_sum(float v, float* sh) {
  v = lanes_sum<LPR>(v);
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[wave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) v += sh[i];
  }
  return v;
}

// WPR > 1: one row per block of WPR waves; else 256 / LPR rows per block
template <typename T, typename W, int NV, int LPR, int WPR>
__global__ __launch_bounds__(WPR > 1 ? 64 * WPR : 256) void ln_fwd_kernel(
    const T* __restrict__ x, long long ldx, const W* __restrict__ w, const W* __restrict__ b, T* __restrict__ y,
    long long ldy, float* __restrict__ mean, float* __restrict__ rstd, long long rows, int C, float eps) {
  constexpr int V = TokType<T>::V, GS = LPR * WPR;
  __shared__ float sh[WPR > 1 ? WPR : 1];
  const int l = threadIdx.x % GS;
  const long long row = (long long)blockIdx.x * (blockDim.x / GS) + threadIdx.x / GS;
  if (row >= rows) return;                                        // (WPR > 1: one row per block, uniform)
  const T* xr = x + row * ldx;
  float f[NV][V];
  float s = 0.f;
  TokVec<T, V> raw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * GS + l) * V;
    raw[j] = tok_raw_n<T, V>(xr + c, C - c);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    tok_up(raw[j], f[j]);
#pragma unroll
    for (int i = 0; i < V; ++i) s += f[j][i];
  }
  const float mu = group_sum<LPR, WPR>(s, sh) / (float)C;
  s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int n = C - (j * GS + l) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f[j][i] -= mu;
      if (i < n) s += f[j][i] * f[j][i];
    }
  }
  const float rs = 1.f / sqrtf(group_sum<LPR, WPR>(s, sh) / (float)C + eps);
  if (l == 0) {
    if (mean) mean[row] = mu;
    if (rstd) rstd[row] = rs;
  }
  T* yr = y + row * ldy;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * GS + l) * V, n = C - c;
    float o[V], t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = f[j][i] * rs;
    if (w) {
      tok_load_n<W, V>(w + c, n, t);
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] *= t[i];
    }
    if (b) {
      tok_load_n<W, V>(b + c, n, t);
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] += t[i];
    }
    tok_store_n<T, V>(yr + c, n, o);
  }
}

// part: [gridDim.x][2][C] sums of (dy xh) and dy over the block's rows, or NULL
template <typename T, typename W, int NV, int LPR, int WPR>
__global__ __launch_bounds__(WPR > 1 ? 64 * WPR : 256) void ln_bwd_kernel(
    const T* __restrict__ dy, long long lddy, const T* __restrict__ x, long long ldx, const W* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, long long lddx,
    float* __restrict__ part, long long rows, int C) {
  constexpr int V = TokType<T>::V, GS = LPR * WPR, NT = WPR > 1 ? 64 * WPR : 256, NG = NT / GS;
  __shared__ float sh[2 * (WPR > 1 ? WPR : 1)];
  __shared__ float cols[WPR > 1 ? 1 : NT * V * NV];
  const int l = threadIdx.x % GS, grp = threadIdx.x / GS;
  float wv[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * GS + l) * V;
    if (w) tok_load_n<W, V>(w + c, C - c, wv[j]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!w) wv[j][i] = 1.f;
      aw[j][i] = ab[j][i] = 0.f;
    }
  }
  const float invC = 1.f / (float)C;
  for (long long r0 = (long long)blockIdx.x * NG; r0 < rows; r0 += (long long)gridDim.x * NG) {
    const long long row = r0 + grp;
    const bool live = row < rows;
    const T* xr = x + row * ldx;
    const T* gr = dy + row * lddy;
    const float mu = live ? mean[row] : 0.f, rs = live ? rstd[row] : 0.f;
    float xh[NV][V], g[NV][V], s1 = 0.f, s2 = 0.f;
    TokVec<T, V> rx[NV], rg[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * GS + l) * V, n = live ? C - c : 0;
      rx[j] = tok_raw_n<T, V>(xr + c, n);
      rg[j] = tok_raw_n<T, V>(gr + c, n);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      tok_up(rx[j], xh[j]);
      tok_up(rg[j], g[j]);
      const int n = C - (j * GS + l) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[j][i] = i < n ? (xh[j][i] - mu) * rs : 0.f;            // (past the end dy is 0, but mu rs may be infinite)
        aw[j][i] += g[j][i] * xh[j][i];
        ab[j][i] += g[j][i];
        g[j][i] *= wv[j][i];
        s1 += g[j][i];
        s2 += g[j][i] * xh[j][i];
      }
    }
    if constexpr (WPR > 1) {                                       // both sums through one exchange
      s1 = lanes_sum<LPR>(s1);
      s2 = lanes_sum<LPR>(s2);
      const int wave = threadIdx.x >> 6;
      __syncthreads();
      if ((threadIdx.x & 63) == 0) { sh[wave] = s1; sh[WPR + wave] = s2; }
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) { s1 += sh[i]; s2 += sh[WPR + i]; }
    } else {
      s1 = lanes_sum<LPR>(s1);
      s2 = lanes_sum<LPR>(s2);
    }
    s1 *= invC;
    s2 *= invC;
    T* dr = dx + row * lddx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * GS + l) * V, n = live ? C - c : 0;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = rs * (g[j][i] - s1 - xh[j][i] * s2);
      tok_store_n<T, V>(dr + c, n, o);
    }
  }
  if (!part) return;
  float* pw = part + (long long)blockIdx.x * 2 * C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if constexpr (WPR > 1) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * GS + l) * V;
        tok_store_n<float, V>(pw + (long long)which * C + c, C - c, which ? ab[j] : aw[j]);
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) cols[grp * (GS * V * NV) + (j * GS + l) * V + i] = which ? ab[j][i] : aw[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += NT) {
        float s = 0.f;
#pragma unroll 8
        for (int q = 0; q < NG; ++q) s += cols[q * (GS * V * NV) + c];
        pw[(long long)which * C + c] = s;
      }
    }
  }
}

// rows too wide for the register kernels: a block per row, the row read once per pass (it stays in the caches)
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_fwd_wide_kernel(const T* __restrict__ x, long long ldx, const W* __restrict__ w,
                                                           const W* __restrict__ b, T* __restrict__ y, long long ldy,
                                                           float* __restrict__ mean, float* __restrict__ rstd, int C,
                                                           float eps) {
  constexpr int V = TokType<T>::V;
  __shared__ float sh[16];
  const long long row = blockIdx.x;
  const T* xr = x + row * ldx;
  float f[V], t[V], s = 0.f;
  for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
    tok_load_n<T, V>(xr + c, C - c, f);
#pragma unroll
    for (int i = 0; i < V; ++i) s += f[i];
  }
  const float mu = group_sum<64, 16>(s, sh) / (float)C;
  s = 0.f;
  for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
    tok_load_n<T, V>(xr + c, C - c, f);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < C) s += (f[i] - mu) * (f[i] - mu);
  }
  const float rs = 1.f / sqrtf(group_sum<64, 16>(s, sh) / (float)C + eps);
  if (threadIdx.x == 0) {
    if (mean) mean[row] = mu;
    if (rstd) rstd[row] = rs;
  }
  for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
    tok_load_n<T, V>(xr + c, C - c, f);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (f[i] - mu) * rs;
    if (w) {
      tok_load_n<W, V>(w + c, C - c, t);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= t[i];
    }
    if (b) {
      tok_load_n<W, V>(b + c, C - c, t);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] += t[i];
    }
    tok_store_n<T, V>(y + row * ldy + c, C - c, f);
  }
}
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_bwd_wide_kernel(const T* __restrict__ dy, long long lddy,
                                                           const T* __restrict__ x, long long ldx,
                                                           const W* __restrict__ w, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, T* __restrict__ dx,
                                                           long long lddx, int C) {
  constexpr int V = TokType<T>::V;
  __shared__ float sh[16];
  const long long row = blockIdx.x;
  const float mu = mean[row], rs = rstd[row];
  float f[V], g[V], t[V], s1 = 0.f, s2 = 0.f;
  auto load = [&](int c) {
    tok_load_n<T, V>(x + row * ldx + c, C - c, f);
    tok_load_n<T, V>(dy + row * lddy + c, C - c, g);
    if (w) tok_load_n<W, V>(w + c, C - c, t);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      f[i] = c + i < C ? (f[i] - mu) * rs : 0.f;
      if (w) g[i] *= t[i];
    }
  };
  for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
    load(c);
#pragma unroll
    for (int i = 0; i < V; ++i) { s1 += g[i]; s2 += g[i] * f[i]; }
  }
  s1 = group_sum<64, 16>(s1, sh) / (float)C;
  s2 = group_sum<64, 16>(s2, sh) / (float)C;
  for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
    load(c);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = rs * (g[i] - s1 - f[i] * s2);
    tok_store_n<T, V>(dx + row * lddx + c, C - c, f);
  }
}
// the weight's partial sums for wide rows: a thread per column, gridDim.y slices of the rows
template <typename T>
__global__ __launch_bounds__(256) void ln_dw_wide_kernel(const T* __restrict__ dy, long long lddy,
                                                         const T* __restrict__ x, long long ldx,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         float* __restrict__ part, long long rows, int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float aw = 0.f, ab = 0.f;
  for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = TokType<T>::up(dy[r * lddy + c]);
    aw += g * (TokType<T>::up(x[r * ldx + c]) - mean[r]) * rstd[r];
    ab += g;
  }
  part[(long long)blockIdx.y * 2 * C + c] = aw;
  part[(long long)blockIdx.y * 2 * C + C + c] = ab;
}

// dw, db = sums of the partial rows: 32 columns by 32 slices of the rows per block, the slices joined in LDS
template <typename W>
__global__ __launch_bounds__(1024) void ln_finish_kernel(const float* __restrict__ part, int nparts, int C,
                                                         W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float sh[32][33];
  const int lc = threadIdx.x & 31, q = threadIdx.x >> 5, c = blockIdx.x * 32 + lc;   // c over [dw | db]
  float s = 0.f;
  if (c < 2 * C) {
#pragma unroll 8
    for (int r = q; r < nparts; r += 32) s += part[(long long)r * 2 * C + c];
  }
  sh[q][lc] = s;
  __syncthreads();
  if (q == 0 && c < 2 * C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sh[i][lc];
    if (c < C) {
      if (dw) dw[c] = TokType<W>::down(s);
    } else if (db) {
      db[c - C] = TokType<W>::down(s);
    }
  }
}

// blocks of the backward kernel, each of which leaves a partial row: what the registers let the chip hold (16 waves per CU
// up to two chunks per lane, 8 above)
#define LN_MAX_PARTS(nv) ((nv) == 1 || (nv) == 2 ? 1024 : 512)
// rows a block of the backward kernel takes at a time, and whether the register kernels hold the row
struct LnPlan { int nv, lpr, wpr; };
static LnPlan ln_plan(int type, int C) {
  const int V = type == RIED_T_F32 ? 4 : 8, chunks = ceil_div(C, V);
  if (chunks <= 8) return {1, 8, 1};
  if (chunks <= 16) return {1, 16, 1};
  if (chunks <= 32) return {1, 32, 1};
  if (chunks <= 64) return {1, 64, 1};
  if (chunks <= 128) return {2, 64, 1};
  if (chunks <= 256) return {4, 64, 1};
  if (chunks <= 512) return {2, 64, 4};
  if (chunks <= 1024) return {4, 64, 4};
  if (chunks <= 2048) return {2, 64, 16};                       // (wider in registers would spill at 16 waves)
  return {0, 0, 0};
}
#define LN_PLANS(M)                                                                                                  \
  if (pl.nv == 1 && pl.lpr == 8) { M(1, 8, 1) }                                                                      \
  else if (pl.nv == 1 && pl.lpr == 16) { M(1, 16, 1) }                                                               \
  else if (pl.nv == 1 && pl.lpr == 32) { M(1, 32, 1) }                                                               \
  else if (pl.nv == 1) { M(1, 64, 1) }                                                                               \
  else if (pl.nv == 2 && pl.wpr == 1) { M(2, 64, 1) }                                                                \
  else if (pl.wpr == 1) { M(4, 64, 1) }                                                                              \
  else if (pl.wpr == 16) { M(2, 64, 16) }                                                                            \
  else if (pl.nv == 2) { M(2, 64, 4) }                                                                               \
  else { M(4, 64, 4) }

static int ln_parts(long long rows, int type, int C) {
  const LnPlan pl = ln_plan(type, C);
  const long long per = pl.nv == 0 ? 64 : pl.wpr > 1 ? 1 : 256 / pl.lpr;
  long long n = (rows + per - 1) / per;
  const int most = pl.wpr > 1 ? LN_MAX_PARTS(pl.nv) / pl.wpr * 2 : LN_MAX_PARTS(pl.nv);
  return (int)(n > most ? most : n);
}

extern "C" long long ried_layer_norm_bwd_scratch_floats(long long rows, int C, int type) {
  if (rows <= 0 || C <= 0 || !tok_type_ok(type)) return 0;
  return (long long)ln_parts(rows, type, C) * 2 * C;
}

// element type T of the rows, W of the parameters
#define LN_DISPATCH(...)                                              \
  TOK_DISPATCH(type, T, {                                             \
    if (wtype == RIED_T_F32) { using W = float; __VA_ARGS__; }        \
    else { using W = T; __VA_ARGS__; }                                \
  })
#define LN_CHECK(name)                                                                                               \
  RIED_CHECK_ARG(rows >= 0 && C > 0 && C <= (1 << 24), name ": bad sizes (%lld rows of %d)", rows, C);               \
  RIED_CHECK_ARG(tok_type_ok(type) && (wtype == RIED_T_F32 || wtype == type),                                        \
                 name ": types are 0 fp32, 1 bf16, 2 fp16; parameters are fp32 or of the rows' type");               \
  const LnPlan pl = ln_plan(type, C);                                                                                 \
  RIED_CHECK_ARG(rows < (1ll << 32) / (pl.nv == 0 ? 1024 : pl.lpr * pl.wpr) - 256, name ": too many rows (%lld)", rows)

extern "C" int ried_layer_norm_fwd(const void* x, long long ldx, const void* w, const void* b, void* y, long long ldy,
                                   float* mean, float* rstd, long long rows, int C, float eps, int type, int wtype,
                                   hipStream_t stream) {
  LN_CHECK("ried_layer_norm_fwd");
  if (rows == 0) return RIED_OK;
  RIED_CHECK_ARG(x && y, "ried_layer_norm_fwd: null pointer");
  RIED_CHECK_ARG(ldx >= C && ldy >= C, "ried_layer_norm_fwd: rows overlap (ldx %lld, ldy %lld, %d columns)", ldx, ldy, C);
  LN_DISPATCH({
#define LN_FWD(NV, LPR, WPR)                                                                                         \
  hipLaunchKernelGGL((ln_fwd_kernel<T, W, NV, LPR, WPR>), dim3(ceil_div(rows, WPR > 1 ? 1 : 256 / LPR)),             \
                     dim3(WPR > 1 ? 64 * WPR : 256), 0, stream, (const T*)x, ldx, (const W*)w, (const W*)b, (T*)y,   \
                     ldy, mean, rstd, rows, C, eps);
    if (pl.nv == 0)
      hipLaunchKernelGGL((ln_fwd_wide_kernel<T, W>), dim3((unsigned)rows), dim3(1024), 0, stream, (const T*)x, ldx,
                         (const W*)w, (const W*)b, (T*)y, ldy, mean, rstd, C, eps);
    else LN_PLANS(LN_FWD)
  });
  RIED_CHECK_LAUNCH("ried_layer_norm_fwd");
  return RIED_OK;
}

extern "C" int ried_layer_norm_bwd(const void* dy, long long lddy, const void* x, long long ldx, const void* w,
                                   const float* mean, const float* rstd, void* dx, long long lddx, void* dw, void* db,
                                   float* scratch, long long rows, int C, int type, int wtype, hipStream_t stream) {
  LN_CHECK("ried_layer_norm_bwd");
  RIED_CHECK_ARG(rows == 0 || (dy && x && mean && rstd && dx), "ried_layer_norm_bwd: null pointer");
  RIED_CHECK_ARG(rows == 0 || (lddy >= C && ldx >= C && lddx >= C), "ried_layer_norm_bwd: rows overlap");
  RIED_CHECK_ARG(!(dw || db) || scratch || rows == 0,
                 "ried_layer_norm_bwd: parameter gradients need ried_layer_norm_bwd_scratch_floats() of scratch");
  const bool sums = dw || db;
  const int nparts = rows > 0 ? ln_parts(rows, type, C) : 0;
  if (rows > 0) {
    LN_DISPATCH({
#define LN_BWD(NV, LPR, WPR)                                                                                         \
  hipLaunchKernelGGL((ln_bwd_kernel<T, W, NV, LPR, WPR>), dim3(nparts), dim3(WPR > 1 ? 64 * WPR : 256), 0, stream,   \
                     (const T*)dy, lddy, (const T*)x, ldx, (const W*)w, mean, rstd, (T*)dx, lddx,                    \
                     sums ? scratch : nullptr, rows, C);
      if (pl.nv == 0) {
        hipLaunchKernelGGL((ln_bwd_wide_kernel<T, W>), dim3((unsigned)rows), dim3(1024), 0, stream, (const T*)dy, lddy,
                           (const T*)x, ldx, (const W*)w, mean, rstd, (T*)dx, lddx, C);
        if (sums)
          hipLaunchKernelGGL((ln_dw_wide_kernel<T>), dim3(ceil_div(C, 256), nparts), dim3(256), 0, stream, (const T*)dy,
                             lddy, (const T*)x, ldx, mean, rstd, scratch, rows, C);
      } else LN_PLANS(LN_BWD)
    });
  }
  if (sums) {                                                      // (no rows: the sums are zeros)
    TOK_DISPATCH(wtype, W, hipLaunchKernelGGL((ln_finish_kernel<W>), dim3(ceil_div(2ll * C, 32)), dim3(1024), 0, stream,
                                              scratch, nparts, C, (W*)dw, (W*)db));
  }
  RIED_CHECK_LAUNCH("ried_layer_norm_bwd");
  return RIED_OK;
}
