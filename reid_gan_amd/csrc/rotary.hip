// Rotary positions of several axes (slice, row, column of a volume): pair j of a token's vector belongs to axis a(j) and
// is turned by the angle t = position[a(j)] * f[j]:  (x0, x1) -> (x0 cos t - x1 sin t, x1 cos t + x0 sin t).
// HBM-bound: every element is read and written once.  The angles are formed once per (token, pair) for all heads, in 64
// bits - a 32-bit product of a far position and a frequency of 1 is off by 2^-24 of the position, in radians - reduced to
// a part of a turn and passed on as 32-bit cosines and sines through LDS.  The backward pass is the turn by -t.
// Measured, 65536 tokens of 16 x 64 channels in bf16: 45 us for 269 MB (6.0 TB/s: part of it stays in the last cache; a copy
// of 256 MB runs at 5.4).  With one chunk in flight per thread, 64-bit divisions and the table read by elements it took 86.
// 64 tokens of 32 x 128: 3.6 us.
#include "tokens.h"

#define ROT_MAX_PAIRS 256
#define ROT_TABLE 2048       // (token, pair) entries per block: 16 KB of LDS
#define ROT_UNROLL 4         // chunks of 16 + 16 bytes a thread has in flight

struct RotArgs {
  const void* x;
  void* y;
  const void* pos;
  const double* freqs;
  long long xb, xl, xh, yb, yl, yh, pb, pl, pa;
  int L, H, D, pairs, s1, s2, s3, tpb, lblocks, chunks;
  int ptype;                 // 0 int32, 1 int64, 2 fp32
  float sign, inv_pairs, inv_per, inv_chunks;
};

// WHOLE: the pairs are whole chunks, no load or store needs a bound
template <typename T, bool INTER, bool WHOLE>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs A) {
  constexpr int V = TokType<T>::V;                               // pairs per chunk
  __shared__ __align__(16) float cs[ROT_TABLE], sn[ROT_TABLE];   // rows of `pitch` entries: whole chunks, read 16 bytes at a time
  const int b = blockIdx.x / A.lblocks, l0 = (blockIdx.x - b * A.lblocks) * A.tpb;
  const int nt = A.L - l0 < A.tpb ? A.L - l0 : A.tpb, pitch = A.chunks * V;
  for (int i = threadIdx.x; i < nt * A.pairs; i += 256) {
    int j;
    const int t = fast_div(i, A.pairs, A.inv_pairs, j);
    const long long at = b * A.pb + (long long)(l0 + t) * A.pl + ((j >= A.s1) + (j >= A.s2) + (j >= A.s3)) * A.pa;
    const double p = A.ptype == 0 ? (double)((const int*)A.pos)[at]
                   : A.ptype == 1 ? (double)((const long long*)A.pos)[at] : (double)((const float*)A.pos)[at];
    double turns = p * (A.freqs[j] * 0.15915494309189533577);
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    cs[t * pitch + j] = c;
    sn[t * pitch + j] = s * A.sign;
  }
  __syncthreads();
  const T* xb = (const T*)A.x + b * A.xb + l0 * A.xl;
  T* yb = (T*)A.y + b * A.yb + l0 * A.yl;
  const int per = A.H * A.chunks, all = nt * per;
  // A thread's chunks: loaded together, then turned and stored (in place a chunk is read before it is written, and no
  // other thread's)
  for (int i0 = threadIdx.x; i0 < all; i0 += 256 * ROT_UNROLL) {
    TokVec<T, V> a[ROT_UNROLL], c[ROT_UNROLL];
    int n[ROT_UNROLL], tab[ROT_UNROLL];
    T* yp[ROT_UNROLL];
#pragma unroll
    for (int u = 0; u < ROT_UNROLL; ++u) {
      const int i = i0 + u * 256 < all ? i0 + u * 256 : i0;
      int r, j;
      const int t = fast_div(i, per, A.inv_per, r), h = fast_div(r, A.chunks, A.inv_chunks, j);
      j *= V;
      n[u] = i0 + u * 256 < all ? (WHOLE ? V : A.pairs - j) : 0;
      tab[u] = t * pitch + j;
      const T* xp = xb + t * A.xl + h * A.xh;
      yp[u] = yb + t * A.yl + h * A.yh;
      if constexpr (INTER) {
        xp += 2 * j;
        yp[u] += 2 * j;
        a[u] = WHOLE ? tok_raw<T, V>(xp) : tok_raw_n<T, V>(xp, 2 * n[u]);
        c[u] = WHOLE ? tok_raw<T, V>(xp + V) : tok_raw_n<T, V>(xp + V, 2 * n[u] - V);
      } else {
        xp += j;
        yp[u] += j;
        a[u] = WHOLE ? tok_raw<T, V>(xp) : tok_raw_n<T, V>(xp, n[u]);
        c[u] = WHOLE ? tok_raw<T, V>(xp + A.pairs) : tok_raw_n<T, V>(xp + A.pairs, n[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < ROT_UNROLL; ++u) {
      if (WHOLE && n[u] == 0) break;                             // (n is V, or 0 from here on)
      float tc[V], ts[V], p[V], q[V], x0[V], x1[V];
      tok_up(a[u], x0);
      tok_up(c[u], x1);
#pragma unroll
      for (int k = 0; k < V; k += 4) {
        const f32x4 c4 = *reinterpret_cast<const f32x4*>(cs + tab[u] + k), s4 = *reinterpret_cast<const f32x4*>(sn + tab[u] + k);
#pragma unroll
        for (int e = 0; e < 4; ++e) { tc[k + e] = c4[e]; ts[k + e] = s4[e]; }
      }
      if constexpr (INTER) {
#pragma unroll
        for (int k = 0; k < V / 2; ++k) {
          p[2 * k] = x0[2 * k] * tc[k] - x0[2 * k + 1] * ts[k];
          p[2 * k + 1] = x0[2 * k + 1] * tc[k] + x0[2 * k] * ts[k];
          q[2 * k] = x1[2 * k] * tc[k + V / 2] - x1[2 * k + 1] * ts[k + V / 2];
          q[2 * k + 1] = x1[2 * k + 1] * tc[k + V / 2] + x1[2 * k] * ts[k + V / 2];
        }
        if (WHOLE) tok_store<T, V>(yp[u], p);
        else tok_store_n<T, V>(yp[u], 2 * n[u], p);
        if (WHOLE) tok_store<T, V>(yp[u] + V, q);
        else tok_store_n<T, V>(yp[u] + V, 2 * n[u] - V, q);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          p[k] = x0[k] * tc[k] - x1[k] * ts[k];
          q[k] = x1[k] * tc[k] + x0[k] * ts[k];
        }
        if (WHOLE) tok_store<T, V>(yp[u], p);
        else tok_store_n<T, V>(yp[u], n[u], p);
        if (WHOLE) tok_store<T, V>(yp[u] + A.pairs, q);
        else tok_store_n<T, V>(yp[u] + A.pairs, n[u], q);
      }
    }
  }
  // channels behind the rotated ones pass through
  const int rest = A.D - 2 * A.pairs;
  if (rest > 0 && A.x != (const void*)A.y) {
    for (int i = threadIdx.x; i < nt * A.H * rest; i += 256) {
      const int t = i / (A.H * rest), r = i - t * (A.H * rest), h = r / rest, d = 2 * A.pairs + r - h * rest;
      yb[t * A.yl + h * A.yh + d] = xb[t * A.xl + h * A.xh + d];
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
  A.L = L; A.H = H; A.D = D; A.pairs = pairs; A.ptype = pos_type;
  A.s1 = s0; A.s2 = s0 + s1; A.s3 = s0 + s1 + s2;
  A.sign = inverse ? -1.f : 1.f;
  const int V = type == RIED_T_F32 ? 4 : 8;
  A.chunks = ceil_div(pairs, V);
  RIED_CHECK_ARG((long long)H * D < (1ll << 20), "ried_rotary: %d heads of %d channels are too many", H, D);
  // a block takes about 1024 chunks (one round of four per thread) of one batch entry, as many tokens as the table holds, and
  // leaves 512 blocks to the chip
  long long tpb = ceil_div(1024, H * A.chunks);
  if (tpb > ROT_TABLE / (A.chunks * V)) tpb = ROT_TABLE / (A.chunks * V);
  const long long most = ((long long)B * L + 511) / 512;
  if (tpb > most) tpb = most;
  A.tpb = (int)(tpb < 1 ? 1 : tpb);
  A.lblocks = ceil_div(L, A.tpb);
  A.inv_pairs = 1.f / (float)pairs;
  A.inv_per = 1.f / (float)(H * A.chunks);
  A.inv_chunks = 1.f / (float)A.chunks;
  const long long blocks = (long long)B * A.lblocks;
  RIED_CHECK_ARG(blocks < (1ll << 24), "ried_rotary: too many tokens");
  TOK_DISPATCH(type, T, {
#define ROT_LAUNCH(INTER, WHOLE) hipLaunchKernelGGL((rotary_kernel<T, INTER, WHOLE>), dim3((unsigned)blocks), dim3(256), 0, stream, A)
    if (pairs % V == 0) { if (interleaved) ROT_LAUNCH(true, true); else ROT_LAUNCH(false, true); }
    else { if (interleaved) ROT_LAUNCH(true, false); else ROT_LAUNCH(false, false); }
  });
  RIED_CHECK_LAUNCH("ried_rotary");
  return RIED_OK;
}
