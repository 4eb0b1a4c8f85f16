// Rotary positions of several axes (slice, row, column of a volume): pair j of a token's vector belongs to axis a(j) and
// is turned by the angle t = position[a(j)] * f[j]:  (x0, x1) -> (x0 cos t - x1 sin t, x1 cos t + x0 sin t).
// HBM-bound: every element is read and written once.  The angles are formed once per (token, pair) for all heads, in 64
// bits - a 32-bit product of a far position and a frequency of 1 is off by 2^-24 of the position, in radians - reduced to
// a part of a turn and passed on as 32-bit cosines and sines through LDS.  The backward pass is the turn by -t.
#include "tokens.h"

#define ROT_MAX_PAIRS 256
#define ROT_TABLE 2048       // (token, pair) entries per block: 16 KB of LDS

struct RotArgs {
  const void* x;
  void* y;
  const void* pos;
  const double* freqs;
  long long xb, xl, xh, yb, yl, yh, pb, pl, pa;
  long long tokens;
  int L, H, D, pairs, s1, s2, s3, tpb, chunks;
  int ptype;                 // 0 int32, 1 int64, 2 fp32
  float sign;
};

template <typename T, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs A) {
  constexpr int V = TokType<T>::V;
  __shared__ float cs[ROT_TABLE], sn[ROT_TABLE];
  const long long t0 = (long long)blockIdx.x * A.tpb;
  const int nt = A.tokens - t0 < A.tpb ? (int)(A.tokens - t0) : A.tpb;
  for (int i = threadIdx.x; i < nt * A.pairs; i += 256) {
    const int t = i / A.pairs, j = i - t * A.pairs;
    const long long tok = t0 + t, b = tok / A.L, l = tok - b * A.L;
    const long long at = b * A.pb + l * A.pl + ((j >= A.s1) + (j >= A.s2) + (j >= A.s3)) * A.pa;
    const double p = A.ptype == 0 ? (double)((const int*)A.pos)[at]
                   : A.ptype == 1 ? (double)((const long long*)A.pos)[at] : (double)((const float*)A.pos)[at];
    double turns = p * (A.freqs[j] * 0.15915494309189533577);
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    cs[i] = c;
    sn[i] = s * A.sign;
  }
  __syncthreads();
  const int per = A.H * A.chunks;
  for (int i = threadIdx.x; i < nt * per; i += 256) {
    const int t = i / per, r = i - t * per, h = r / A.chunks, j = (r - h * A.chunks) * V;   // pairs j .. j + V - 1
    const long long tok = t0 + t, b = tok / A.L, l = tok - b * A.L;
    const T* xp = (const T*)A.x + b * A.xb + l * A.xl + h * A.xh;
    T* yp = (T*)A.y + b * A.yb + l * A.yl + h * A.yh;
    const int n = A.pairs - j;
    const float* tc = cs + t * A.pairs + j;
    const float* ts = sn + t * A.pairs + j;
    float a[V], c[V], p[V], q[V];
    if constexpr (INTER) {
      tok_load_n<T, V>(xp + 2 * j, 2 * n, a);
      tok_load_n<T, V>(xp + 2 * j + V, 2 * n - V, c);
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        if (k < n) {
          p[2 * k] = a[2 * k] * tc[k] - a[2 * k + 1] * ts[k];
          p[2 * k + 1] = a[2 * k + 1] * tc[k] + a[2 * k] * ts[k];
        }
        if (k + V / 2 < n) {
          q[2 * k] = c[2 * k] * tc[k + V / 2] - c[2 * k + 1] * ts[k + V / 2];
          q[2 * k + 1] = c[2 * k + 1] * tc[k + V / 2] + c[2 * k] * ts[k + V / 2];
        }
      }
      tok_store_n<T, V>(yp + 2 * j, 2 * n, p);
      tok_store_n<T, V>(yp + 2 * j + V, 2 * n - V, q);
    } else {
      tok_load_n<T, V>(xp + j, n, a);
      tok_load_n<T, V>(xp + A.pairs + j, n, c);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (k < n) {
          p[k] = a[k] * tc[k] - c[k] * ts[k];
          q[k] = c[k] * tc[k] + a[k] * ts[k];
        }
      }
      tok_store_n<T, V>(yp + j, n, p);
      tok_store_n<T, V>(yp + A.pairs + j, n, q);
    }
  }
  // channels behind the rotated ones pass through
  const int rest = A.D - 2 * A.pairs;
  if (rest > 0 && A.x != (const void*)A.y) {
    for (int i = threadIdx.x; i < nt * A.H * rest; i += 256) {
      const int t = i / (A.H * rest), r = i - t * (A.H * rest), h = r / rest, d = 2 * A.pairs + r - h * rest;
      const long long tok = t0 + t, b = tok / A.L, l = tok - b * A.L;
      ((T*)A.y)[b * A.yb + l * A.yl + h * A.yh + d] = ((const T*)A.x)[b * A.xb + l * A.xl + h * A.xh + d];
    }
  }
}

extern "C" int ried_rotary(const void* x, long long xb, long long xl, long long xh, void* y, long long yb, long long yl,
                           long long yh, const void* pos, int pos_type, long long pb, long long pl, long long pa,
                           const double* freqs, int s0, int s1, int s2, int s3, int B, int L, int H, int D,
                           int interleaved, int inverse, int type, hipStream_t stream) {
  RIED_CHECK_ARG(B >= 0 && L >= 0 && H > 0 && D > 0 && H <= 65536 && D <= 65536, "ried_rotary: bad sizes (%d, %d, %d, %d)", B, L, H, D);
  RIED_CHECK_ARG(tok_type_ok(type) && pos_type >= 0 && pos_type <= 2, "ried_rotary: bad element or position type");
  RIED_CHECK_ARG(s0 >= 0 && s1 >= 0 && s2 >= 0 && s3 >= 0 && s0 <= D && s1 <= D && s2 <= D && s3 <= D, "ried_rotary: bad sections");
  const int pairs = s0 + s1 + s2 + s3;
  RIED_CHECK_ARG(pairs > 0 && 2 * pairs <= D && pairs <= ROT_MAX_PAIRS,
                 "ried_rotary: %d pairs do not fit %d channels (at most %d pairs)", pairs, D, ROT_MAX_PAIRS);
  if (B == 0 || L == 0) return RIED_OK;
  RIED_CHECK_ARG(x && y && pos && freqs, "ried_rotary: null pointer");
  RIED_CHECK_ARG(x != y || (xb == yb && xl == yl && xh == yh), "ried_rotary: in place needs equal strides");
  RotArgs A;
  A.x = x; A.y = y; A.pos = pos; A.freqs = freqs;
  A.xb = xb; A.xl = xl; A.xh = xh; A.yb = yb; A.yl = yl; A.yh = yh; A.pb = pb; A.pl = pl; A.pa = pa;
  A.tokens = (long long)B * L;
  A.L = L; A.H = H; A.D = D; A.pairs = pairs; A.ptype = pos_type;
  A.s1 = s0; A.s2 = s0 + s1; A.s3 = s0 + s1 + s2;
  A.sign = inverse ? -1.f : 1.f;
  const int V = type == RIED_T_F32 ? 4 : 8;
  A.chunks = ceil_div(pairs, V);
  // a block takes about 1024 chunks (four per thread), as many tokens as the table holds, and leaves 512 blocks to the chip
  long long tpb = ceil_div(1024, H * A.chunks);
  if (tpb > ROT_TABLE / pairs) tpb = ROT_TABLE / pairs;
  const long long most = (A.tokens + 511) / 512;
  if (tpb > most) tpb = most;
  A.tpb = (int)(tpb < 1 ? 1 : tpb);
  const long long blocks = (A.tokens + A.tpb - 1) / A.tpb;
  RIED_CHECK_ARG(blocks <= 0x7fffffffll, "ried_rotary: too many tokens");
  TOK_DISPATCH(type, T, {
    if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, stream, A);
    else hipLaunchKernelGGL((rotary_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, stream, A);
  });
  RIED_CHECK_LAUNCH("ried_rotary");
  return RIED_OK;
}
