// AdamW (decoupled weight decay) over many tensors in one launch, moments in 32 bits or in 8.
//   t += 1;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// 8-bit moments: blocks of 256 elements share a scale; m is held as e4m3 codes of m * 448 / max|m|, and in place of v its
// root r, as e4m3 codes of r * 448 / max r.  The root halves the exponent range v needs, so e4m3's 17 octaves span 34 of
// v; a positive root never rounds to zero (it takes the smallest code), because a lost v would make the next step
// m / eps.  The step itself uses the unrounded m and r.  Blocks whose largest value is below 2^-100 are stored as zeros;
// a NaN or infinity makes its block's state NaN.
// HBM-bound: 28 bytes per element with fp32 moments and parameters, 6 + 4 with bf16 parameters and 8-bit moments.  A wave
// takes whole blocks of 256 (four elements per lane, four blocks in flight), so a block's maximum is one wave reduction
// in registers.  Every operation on the moments is rounded by itself (no contraction): the codes do not depend on how the
// compiler fuses, and an elementwise evaluation in 32 bits gives the same bits.
// Measured: 222 fp32 tensors of 16 to 524288 elements, 315 MB: 65 us (4.8 TB/s) + 2.6 for the step counts; 48 bf16 tensors of
// up to 16777216 elements with 8-bit moments, 747 MB: 149 to 154 us (4.9 TB/s; a copy of 1 GB runs at 5.1).  All of a
// workgroup's loads are in flight before the first is used: with a branch between them 75 and 179 us.
#include "tokens.h"

#define ADAMW_TENSORS 440    // gradient pointers per launch: they travel as kernel arguments (3.5 of the 4 KB)
#define ADAMW_CHUNK 4096     // elements per workgroup
#define ADAMW_BLOCK 256      // elements that share a scale
#define ADAMW_TOP 448.f
#define ADAMW_FLOOR 0.001953125f

struct AdamwGrads { const void* g[ADAMW_TENSORS]; };
struct AdamwConst { float b1, c1, b2, c2, eps, keep; };
struct AdamwJob { long long p, m, v, ms, vs, n; };       // pointers (ms, vs: scales of the 8-bit moments) and elements

// step counts and the factors that follow from them; tensors without a gradient keep their count
__global__ __launch_bounds__(256) void adamw_tick_kernel(AdamwGrads G, int first, int count, int* __restrict__ steps,
                                                         float* __restrict__ coef, double lr, double b1, double b2) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= count || G.g[i] == nullptr) return;
  const int t = ++steps[first + i];
  coef[2 * (first + i)] = (float)(lr / (1.0 - pow(b1, (double)t)));
  coef[2 * (first + i) + 1] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
}

__device__ __forceinline__ unsigned umax_(unsigned a, unsigned b) { return a > b ? a : b; }
// largest over the wave, in every lane (on the bits of absolute values: NaN above infinity above the rest)
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
  v = umax_(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true));
  v = umax_(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, true));
  v = umax_(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, true));
  v = umax_(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, true));
  unsigned x = v, y = v;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  x = umax_(x, y);
  y = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  return umax_(x, y);
}
__device__ __forceinline__ void from_codes(unsigned u, float scale, float (&f)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
  f[0] = lo[0] * scale; f[1] = lo[1] * scale; f[2] = hi[0] * scale; f[3] = hi[1] * scale;
}
// codes of four values of a block and the block's scale
template <bool POSITIVE>
__device__ __forceinline__ unsigned to_codes(const float (&f)[4], float& scale) {
#pragma clang fp contract(off)
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = umax_(top, __builtin_bit_cast(unsigned, f[i]) & 0x7fffffffu);
  const float mx = __builtin_bit_cast(float, wave_umax(top));
  const bool none = mx < 0x1p-100f;
  scale = none ? 0.f : mx * (float)(1.0 / 448.0);
  const float inv = none ? 0.f : (1.f / mx) * ADAMW_TOP;
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    q[i] = f[i] * inv;
    if (POSITIVE && !none && f[i] > 0.f && q[i] < ADAMW_FLOOR) q[i] = ADAMW_FLOOR;
  }
  int u = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], u, true);
}

// FULL: all elements of the workgroup's chunk exist
template <typename T, bool SMALL, bool FULL>
__device__ __forceinline__ void adamw_body(const AdamwJob& J, const T* __restrict__ g, int chunk, float rate, float root,
                                           const AdamwConst& K) {
#pragma clang fp contract(off)
  T* p = (T*)J.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long e0 = (long long)chunk * ADAMW_CHUNK + wave * 1024;
  TokVec<T, 4> pr[4], gr[4];
  f32x4 mr[4], vr[4];
  unsigned mc[4], rc[4];
  float ms[4], rs[4];
  int n[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const long long at = e0 + k * ADAMW_BLOCK + lane * 4, left = J.n - at, blk = (e0 >> 8) + k;
    n[k] = left > 4 ? 4 : (int)left;
    // (the moments' buffers hold whole blocks of 256: no bound inside a block that exists)
    const bool live = FULL || blk * ADAMW_BLOCK < J.n;
    if constexpr (FULL) {
      pr[k] = tok_raw<T, 4>(p + at);
      gr[k] = tok_raw<T, 4>(g + at);
    } else {
      pr[k] = tok_raw_n<T, 4>(p + at, n[k]);
      gr[k] = tok_raw_n<T, 4>(g + at, n[k]);
    }
    if constexpr (SMALL) {
      mc[k] = rc[k] = 0u;
      ms[k] = rs[k] = 0.f;
      if (live) {
        mc[k] = *(const unsigned*)((const char*)J.m + at);
        rc[k] = *(const unsigned*)((const char*)J.v + at);
        ms[k] = ((const float*)J.ms)[blk];
        rs[k] = ((const float*)J.vs)[blk];
      }
    } else {
      mr[k] = vr[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (live) {
        mr[k] = *(const f32x4*)((const float*)J.m + at);
        vr[k] = *(const f32x4*)((const float*)J.v + at);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const long long at = e0 + k * ADAMW_BLOCK + lane * 4, blk = (e0 >> 8) + k;
    const bool live = FULL || blk * ADAMW_BLOCK < J.n;
    float pv[4], gv[4], m[4], v[4], r[4], o[4];
    tok_up(pr[k], pv);
    tok_up(gr[k], gv);
    if constexpr (SMALL) {
      from_codes(mc[k], ms[k], m);
      from_codes(rc[k], rs[k], r);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = r[i] * r[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) { m[i] = mr[k][i]; v[i] = vr[k][i]; }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = m[i] * K.b1 + gv[i] * K.c1;
      v[i] = v[i] * K.b2 + (gv[i] * gv[i]) * K.c2;
      r[i] = sqrtf(v[i]);
      o[i] = pv[i] * K.keep - rate * (m[i] / (r[i] * root + K.eps));
      if (!FULL && i >= n[k]) m[i] = v[i] = r[i] = 0.f;           // padding of the last block
    }
    if constexpr (SMALL) {
      float sm, sr;
      const unsigned cm = to_codes<false>(m, sm), cr = to_codes<true>(r, sr);
      if (live) {
        *(unsigned*)((char*)J.m + at) = cm;
        *(unsigned*)((char*)J.v + at) = cr;
        if (lane == 0) {
          ((float*)J.ms)[blk] = sm;
          ((float*)J.vs)[blk] = sr;
        }
      }
    } else if (live) {
      *(f32x4*)((float*)J.m + at) = f32x4{m[0], m[1], m[2], m[3]};
      *(f32x4*)((float*)J.v + at) = f32x4{v[0], v[1], v[2], v[3]};
    }
    if constexpr (FULL) tok_store<T, 4>(p + at, o);
    else tok_store_n<T, 4>(p + at, n[k], o);
  }
}

template <typename T, bool SMALL>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwGrads G, const AdamwJob* __restrict__ jobs,
                                                    const int* __restrict__ map, int first, const float* __restrict__ coef,
                                                    AdamwConst K) {
  const int ti = map[2 * blockIdx.x], chunk = map[2 * blockIdx.x + 1];
  const T* g = (const T*)G.g[ti - first];
  if (g == nullptr) return;
  const AdamwJob J = jobs[ti];
  const float rate = coef[2 * ti], root = coef[2 * ti + 1];
  if ((long long)(chunk + 1) * ADAMW_CHUNK <= J.n) adamw_body<T, SMALL, true>(J, g, chunk, rate, root, K);
  else adamw_body<T, SMALL, false>(J, g, chunk, rate, root, K);
}

extern "C" int ried_adamw_jobs(const long long* jobs, const int* map, const long long* grads_host, const int* first_host,
                               int ntensors, int* steps, float* coef, double lr, double b1, double b2, double eps,
                               double weight_decay, int type, int state_bits, hipStream_t stream) {
  RIED_CHECK_ARG(ntensors >= 0 && (ntensors == 0 || (jobs && map && grads_host && first_host && steps && coef)),
                 "ried_adamw_jobs: null pointer");
  RIED_CHECK_ARG(type == RIED_T_F32 || type == RIED_T_BF16, "ried_adamw_jobs: parameters are fp32 (0) or bf16 (1)");
  RIED_CHECK_ARG(state_bits == 32 || state_bits == 8, "ried_adamw_jobs: moments have 32 or 8 bits, not %d", state_bits);
  RIED_CHECK_ARG(lr >= 0 && eps >= 0 && weight_decay >= 0 && b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1,
                 "ried_adamw_jobs: lr, eps and weight_decay are not negative, betas lie in [0, 1)");
  const AdamwConst K = {(float)b1, (float)(1.0 - b1), (float)b2, (float)(1.0 - b2), (float)eps, (float)(1.0 - lr * weight_decay)};
  for (int t0 = 0; t0 < ntensors; t0 += ADAMW_TENSORS) {
    const int cnt = ntensors - t0 < ADAMW_TENSORS ? ntensors - t0 : ADAMW_TENSORS;
    const int b0 = first_host[t0], blocks = first_host[t0 + cnt] - b0;
    AdamwGrads G;
    bool any = false;
    for (int i = 0; i < ADAMW_TENSORS; ++i) {
      G.g[i] = i < cnt ? (const void*)grads_host[t0 + i] : nullptr;
      any |= G.g[i] != nullptr;
    }
    if (!any) continue;
    hipLaunchKernelGGL(adamw_tick_kernel, dim3(ceil_div(cnt, 256)), dim3(256), 0, stream, G, t0, cnt, steps, coef, lr, b1, b2);
    if (blocks <= 0) continue;
#define ADAMW_LAUNCH(T, SMALL)                                                                                         \
  hipLaunchKernelGGL((adamw_kernel<T, SMALL>), dim3(blocks), dim3(256), 0, stream, G, (const AdamwJob*)jobs,           \
                     map + 2 * (long long)b0, t0, coef, K)
    if (type == RIED_T_F32) { if (state_bits == 8) ADAMW_LAUNCH(float, true); else ADAMW_LAUNCH(float, false); }
    else { if (state_bits == 8) ADAMW_LAUNCH(bf16_t, true); else ADAMW_LAUNCH(bf16_t, false); }
  }
  RIED_CHECK_LAUNCH("ried_adamw_jobs");
  return RIED_OK;
}
