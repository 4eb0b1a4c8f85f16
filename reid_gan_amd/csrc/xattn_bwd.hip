// Cross attention, backward:  P = exp(S - lse), Dl = sum_c dO o, dP = dO v^T, dS = P (dP - Dl),
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dO.
// Two kernels, each of which owns what it adds up: rows (dq, over the keys) and keys (dk, dv, over the rows of all heads
// that share them).  The scores are formed twice - 14 D operations a pair instead of 10 D - and in exchange nothing is
// added with atomics: the order of every sum is fixed.
#include "xattn.h"

// Few keys (this many tiles of 64) leave roundings nothing to average out in, so two of them are avoided there.  Dl =
// sum_c dO o = sum_j P dP: the stored o is rounded and was formed from rounded weights, which with two keys is off by as
// much as dP - Dl is large (and with one key dS = 0 is all there is); it is formed from the scores instead, in a first pass
// over the keys.  And what rounding P and dS to the type leaves over enters the products as a second operand.
#define XA_FEW 4
template <typename T> __device__ __forceinline__ u32x4 xa_rest(const f32x16& s, int which, u32x4 rounded) {
  float f[8];
  xa_unpack<T>(rounded, f);
  f32x16 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = s[8 * which + i] - f[i];
  return xa_as_b<T>(r, 0);
}

// s = A f^T and dp += B g^T over 32 rows of two tiles.  The fragments of AHEAD times 16 channels are asked for before their first
// product: left to itself the compiler reads one, waits for it and multiplies (dk and dv of 2 x 16 heads of 128 channels, 2048
// rows by 2048 keys: 263 -> 241 us; of 64 channels, the sizes below: 61 -> 58.5).
template <typename T, int DP, int AHEAD>
__device__ __forceinline__ void xa_scores(const char* a, const char* b, int row, int lane, const u32x4 (&f)[XaTile<DP>::KS],
                                          const u32x4 (&g)[XaTile<DP>::KS], f32x16& s, f32x16& dp) {
  constexpr int KS = XaTile<DP>::KS;
  s = xa_zero();
#pragma unroll
  for (int k0 = 0; k0 < KS; k0 += AHEAD) {
    u32x4 x[AHEAD], y[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (k0 + i < KS) {
        x[i] = xa_frag<DP>(a, row, k0 + i, lane);
        y[i] = xa_frag<DP>(b, row, k0 + i, lane);
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (k0 + i < KS) {
        s = xa_mma<T>(x[i], f[k0 + i], s);
        dp = xa_mma<T>(y[i], g[k0 + i], dp);
      }
  }
}

// fp16 products hold dS only between 2^-24 and 2^16 while P alone spans more: dS travels times a power of two, lowered
// (and the sums with it) when a value would pass 2^15.  bf16 has fp32's range and needs none.
template <typename T> struct XaRange {
  static constexpr bool on = false;
  static constexpr float p_up = 0.f, p_down = 1.f;               // P times 2^p_up; the sums of P times p_down
};
template <> struct XaRange<_Float16> {
  static constexpr bool on = true;
  static constexpr float p_up = 15.f, p_down = 0x1p-15f;
};
template <int DT>
__device__ __forceinline__ void xa_fit(float mx, float& es, f32x16 (&acc)[DT]) {
  if (!__any(mx * es > 32768.f)) return;
  mx = wave_max(mx);
  if (!(mx < INFINITY)) return;
  const float ne = __builtin_amdgcn_exp2f(14.f - ceilf(__log2f(mx))), f = ne / es;
  if (!(ne < es)) return;
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] *= f;
  es = ne;
}

// ---------------------------------------------------------------------------------------------------------------------
// dq: the forward kernel's tiling.  S^T = K Q^T and dP^T = V dO^T per 32 keys, dS^T is the B operand of dq^T += K^T dS^T.
// Measured, 4 x 4096 rows over 657 to 1500 keys, 4 key heads of 64 channels (27 GFLOP): 39.4 us, 690 TFLOP/s; the matrix pipes
// are busy a quarter of the cycles.
// Also leaves for the other kernel what its exponents add (p_up - lse, in powers of two; -infinity for a row without keys)
// and Dl.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void xattn_dq_kernel(XaArgs A) {
  constexpr int KS = XaTile<DP>::KS, DT = XaTile<DP>::DT, RB = XaTile<DP>::RB, NC = XaTile<DP>::NC, RPI = XaTile<DP>::RPI;
  constexpr int TILE = 64 * RB, NI = 16 / RPI;
  extern __shared__ __align__(16) char smem[];                    // [2][K tile, V tile]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  int inner, head;
  xa_block(A.tiles * A.nsplit, A.B * A.Hkv, inner, head);
  const int b = head / A.Hkv, hk = head % A.Hkv, tile = inner % A.tiles, split = inner / A.tiles;
  const int row = tile * 128 + wave * 32 + (lane & 31);
  const bool live = row < A.rows;
  const int g = live ? row / A.Lq : 0, qi = live ? row - g * A.Lq : 0, hq = hk * A.G + g;
  const long long flat = (long long)head * A.rows + row;
  const T* qp = (const T*)A.q + (long long)b * A.qs[0] + (long long)qi * A.qs[1] + (long long)hq * A.qs[2];
  const T* gp = (const T*)A.dout + (long long)b * A.gs[0] + (long long)qi * A.gs[1] + (long long)hq * A.gs[2];
  const T* op = (const T*)A.o + (long long)b * A.os[0] + (long long)qi * A.os[1] + (long long)hq * A.os[2];
  const int nk = xa_keys(A, b), ntile = (nk + 63) >> 6, per = (ntile + A.nsplit - 1) / A.nsplit;
  const int t0 = split * per, t1 = t0 + per < ntile ? t0 + per : ntile;
  const bool few = ntile <= XA_FEW;
  u32x4 fq[KS], fg[KS];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = s * 16 + h * 8;
    const bool ok = live && d < A.D;
    const u32x4 none = {0, 0, 0, 0};
    fq[s] = ok ? *reinterpret_cast<const u32x4*>(qp + d) : none;
    fg[s] = ok ? *reinterpret_cast<const u32x4*>(gp + d) : none;
  }
  if (!few) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = s * 16 + h * 8;
      const u32x4 fo = live && d < A.D ? *reinterpret_cast<const u32x4*>(op + d) : u32x4{0, 0, 0, 0};
      float x[8], y[8];
      xa_unpack<T>(fg[s], x);
      xa_unpack<T>(fo, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) delta += x[i] * y[i];
    }
    float lo, hi;
    xa_halves(delta, lo, hi);
    delta = lo + hi;
  }
  float lse2 = INFINITY;
  if (live) {
    const float l = A.lse[flat];
    lse2 = l == -INFINITY ? INFINITY : l * XA_LOG2E;
  }
  const char* kp = (const char*)((const T*)A.k + (long long)b * A.ks[0] + (long long)hk * A.ks[2]);
  const char* vp = (const char*)((const T*)A.v + (long long)b * A.vs[0] + (long long)hk * A.vs[2]);
  const unsigned char* mp = A.mask ? A.mask + (long long)b * A.ms : nullptr;
  const int krow = (int)A.ks[1] * 2, vrow = (int)A.vs[1] * 2;
  const int srow = wave * RPI + lane / NC, sc = (lane % NC) ^ xa_swz<RB>(srow);
  const unsigned dead = sc * 8 >= A.D ? XA_OOB : 0u;
  const unsigned koff = (unsigned)(srow * krow + sc * 16) | dead, voff = (unsigned)(srow * vrow + sc * 16) | dead;
  auto issue = [&](int t, u64 w, int buf) {
    const __amdgpu_buffer_rsrc_t rk = xa_rsrc(kp + (long long)t * 64 * krow), rv = xa_rsrc(vp + (long long)t * 64 * vrow);
    char* dst = smem + buf * 2 * TILE + wave * RPI * RB;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const unsigned bad = (w >> (srow + i * 4 * RPI)) & 1 ? 0u : XA_OOB;
      xa_dma16(rk, koff | bad, i * 4 * RPI * krow, dst + i * 4 * RPI * RB);
      xa_dma16(rv, voff | bad, i * 4 * RPI * vrow, dst + TILE + i * 4 * RPI * RB);
    }
  };
  auto mask_byte = [&](int t) -> int {
    const int key = t * 64 + lane;
    return mp && key < nk ? mp[key] : 0;
  };
  const float c = A.scale * XA_LOG2E;
  XaTr<DP> tr(smem, lane);
  // tiles f .. e - 1 through the two stages, `use` on each 32 keys of a tile
  auto sweep = [&](int f, int e, const f32x16& start, auto use) {
    u64 w = 0;
    int byte = 0, buf = 0;
    if (f < e) {
      w = xa_word(nk - f * 64, mp != nullptr, mask_byte(f));
      issue(f, w, 0);
      byte = mask_byte(f + 1);
    }
    for (int t = f; t < e; ++t) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      u64 wn = 0;
      if (t + 1 < e) {
        wn = xa_word(nk - (t + 1) * 64, mp != nullptr, byte);
        issue(t + 1, wn, buf ^ 1);
        byte = mask_byte(t + 2);
      }
      if (w) {
        const char* kt = smem + buf * 2 * TILE;
        const char* vt = kt + TILE;
        auto keys32 = [&](auto u_) {
          constexpr int u = decltype(u_)::value;
          f32x16 s, dp = start;
          xa_scores<T, DP, 2>(kt, vt, 32 * u, lane, fq, fg, s, dp);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = xa_exp2(__builtin_fmaf(s[r], c, -lse2));
          if (w != ~0ull) {                                       // (a hidden key's score reads as 0, not as nothing)
            const unsigned bits = (unsigned)(w >> (32 * u)) >> (4 * h);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = (bits >> (8 * (r >> 2) + (r & 3))) & 1 ? s[r] : 0.f;
          }
          use(u_, s, dp);
        };
        keys32(XaInt<0>{}), keys32(XaInt<1>{});
      }
      w = wn;
      tr.move(buf ? -2 * TILE : 2 * TILE);
      buf ^= 1;
    }
    tr.move(buf ? -2 * TILE : 0);
  };
  if (few) {
    sweep(0, ntile, xa_zero(), [&](auto, f32x16& p, f32x16& dp) {
#pragma unroll
      for (int r = 0; r < 16; ++r) delta += p[r] * dp[r];
    });
    float lo, hi;
    xa_halves(delta, lo, hi);
    delta = lo + hi;
    __builtin_amdgcn_s_barrier();                                 // (the stages are free again)
    asm volatile("" ::: "memory");
  }
  if (live && split == 0 && h == 0) {
    A.lse2[flat] = XaRange<T>::p_up - lse2;
    A.delta[flat] = -delta;
  }
  // up to 96 channels the registers hold -Dl as the products' first sum (44.0 -> 42.3 us for the sizes above on one card); above,
  // it is subtracted after them
  constexpr bool FOLD = DP <= 96;
  f32x16 start = xa_zero();
  if constexpr (FOLD) {
#pragma unroll
    for (int r = 0; r < 16; ++r) start[r] = -delta;
  }
  float es = XaRange<T>::on ? 0x1p24f : 1.f;
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = xa_zero();
  auto rows = [&](auto few_) {
    sweep(t0, t1, start, [&](auto u_, f32x16& s, f32x16& dp) {
      constexpr int u = decltype(u_)::value;
      float mx = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] *= FOLD ? dp[r] : dp[r] - delta;
        if constexpr (XaRange<T>::on) mx = fmaxf(mx, fabsf(s[r]));
      }
      if constexpr (XaRange<T>::on) {
        xa_fit<DT>(mx, es, acc);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= es;
      }
      auto add = [&](auto kb_) {
        constexpr int kb = decltype(kb_)::value;
        u32x4 fk[DT];
        xa_tr_frags<DP, u * 32 + kb * 16>(tr, fk);
        const u32x4 f = xa_as_b<T>(s, kb);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = xa_mma<T>(fk[d], f, acc[d]);
        if constexpr (decltype(few_)::value) {
          const u32x4 rest = xa_rest<T>(s, kb, f);
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[d] = xa_mma<T>(fk[d], rest, acc[d]);
        }
      };
      add(XaInt<0>{}), add(XaInt<1>{});
    });
  };
  if (few) rows(XaInt<1>{});
  else rows(XaInt<0>{});
  if (!live) return;
  const float f = A.scale / es;
  if (A.nsplit == 1) {
    T* dst = (T*)A.dq + (long long)b * A.dqs[0] + (long long)qi * A.dqs[1] + (long long)hq * A.dqs[2];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int ch = d * 32 + 2 * r + 4 * h;
        if (ch < A.D)
          *reinterpret_cast<u32x2*>(dst + ch) = u32x2{xa_pack<T>(acc[d][r] * f, acc[d][r + 1] * f),
                                                      xa_pack<T>(acc[d][r + 2] * f, acc[d][r + 3] * f)};
      }
  } else {
    float* dst = A.part + ((long long)split * A.B * A.Hkv * A.rows + flat) * A.D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int ch = d * 32 + 2 * r + 4 * h;
        if (ch < A.D)
          *reinterpret_cast<f32x4*>(dst + ch) = f32x4{acc[d][r] * f, acc[d][r + 1] * f, acc[d][r + 2] * f, acc[d][r + 3] * f};
      }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// dk, dv: a block takes 64 keys at a time and walks tiles of rows (Q, dO and the rows' two numbers through LDS DMA, two
// stages of 128); a wave takes 32 of the keys (K and V fragments in registers) and 64 rows of every tile, and the two row
// groups are added through LDS at the end.  Registers and LDS allow a CU two blocks up to 64 channels, one above.  (Two
// blocks of four waves, each with barriers of its own, against one of eight: 60 against 69 us for 4 x 4096 rows over 657
// to 1500 keys of 4 heads of 64 channels.)  S = Q K^T and dP = dO V^T have the row along the registers, so P and dS are the
// B operands of dv^T += dO^T P and dk^T += Q^T dS as they stand.
//
// The work is (64 keys) x (row tiles) of every batch entry and key head, counted through in that order.  Either a block
// takes one 64 keys with all rows, or the count is dealt out in even shares, one for every block that the chip holds: a share
// begins and ends in the middle of some 64 keys' rows, and leaves those two as partial sums that the next kernel adds, in
// the order of the shares.  With ragged lengths only the 64s that hold keys are counted.  Measured, the sizes above (36 GFLOP):
// 56.4 us, 640 TFLOP/s, + 7.8 for the parts.  (Three blocks per CU, 32 rows a group: the registers spill, 88 us.)  128
// channels, 2 x 16 heads, 2048 rows by 2048 keys (137 GFLOP): 241 us, 570 TFLOP/s: a wave alone on its SIMD runs products
// and the rest one after the other.  (The second 32 rows' scores before the first's exponentials: 250.)
// ---------------------------------------------------------------------------------------------------------------------
template <int DP>
struct XaKv {
  static constexpr int NW = 4, RG = NW / 2, ROWS = 64 * RG, BLOCKS = DP <= 64 ? 2 : 1, STAGE = 2 * ROWS * XaTile<DP>::RB + 8 * ROWS;
};
#define XA_RAGGED 256                                             // batch entries whose lengths are counted
// before[b]: 64s with keys in the batch entries before b
__device__ __forceinline__ void xa_count(const XaArgs& A, int* before) {
  if (!A.ragged) return;
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int n[4], s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      n[i] = lane * 4 + i < A.B ? (xa_keys(A, lane * 4 + i) + 63) >> 6 : 0;
      s += n[i];
    }
    int at = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(at, o, 64);
      if (lane >= o) at += x;
    }
    if (lane == 63) before[XA_RAGGED] = at;
    at -= s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      before[lane * 4 + i] = at;
      at += n[i];
    }
  }
  __syncthreads();
}
// share i of the count is [i * units / n, (i + 1) * units / n); every share has at least two tiles of rows
struct XaShares {
  long long units;
  int per, n;                                                     // row tiles of 64 keys; shares
  __device__ __forceinline__ XaShares(const XaArgs& A, const int* before) {
    per = (A.rows + 127) >> 7;
    units = (long long)(A.ragged ? __builtin_amdgcn_readfirstlane(before[A.B]) : A.B * A.tiles) * A.Hkv * per;
    const long long most = units / 2;
    n = A.nsplit < most ? A.nsplit : most > 0 ? (int)most : units > 0 ? 1 : 0;
  }
  __device__ __forceinline__ long long begin(int i) const { return i * units / n; }
  __device__ __forceinline__ int of(long long unit) const { return (int)(((unit + 1) * n - 1) / units); }
};

template <typename T, int DP>
__global__ __launch_bounds__(64 * XaKv<DP>::NW, XaKv<DP>::BLOCKS) void xattn_dkv_kernel(XaArgs A) {
  constexpr int KS = XaTile<DP>::KS, DT = XaTile<DP>::DT, RB = XaTile<DP>::RB, NC = XaTile<DP>::NC, RPI = XaTile<DP>::RPI;
  constexpr int NW = XaKv<DP>::NW, RG = XaKv<DP>::RG, ROWS = XaKv<DP>::ROWS, TILE = ROWS * RB, STEP = NW * RPI, NI = ROWS / STEP, STAGE = XaKv<DP>::STAGE;
  static_assert(ROWS == 128, "row tiles as they are counted");
  constexpr int EX = 2 * DT * 4 * 64;                             // vectors of four a wave hands over
  static_assert((RG - 1) * 2 * EX * 16 <= 2 * STAGE, "the exchange reuses the stages");
  extern __shared__ __align__(16) char smem[];                    // [2][Q tile, dO tile, ROWS lse2, ROWS Dl]
  __shared__ int before[XA_RAGGED + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int grp = wave >> 1;
  xa_count(A, before);
  long long unit, end;
  int per, share = 0;
  if (A.nsplit == 0) {                                            // a block, a head's 64 keys
    int inner, head;
    xa_block(A.tiles, A.B * A.Hkv, inner, head);
    per = (A.rows + 127) >> 7;
    unit = ((long long)head * A.tiles + inner) * per;
    end = unit + per;
  } else {
    const XaShares S(A, before);
    const int id = blockIdx.x, n = gridDim.x;
    share = (n & 7) == 0 ? (id & 7) * (n >> 3) + (id >> 3) : id;  // (neighbours on one XCD)
    if (share >= S.n) return;
    per = S.per;
    unit = S.begin(share);
    end = S.begin(share + 1);
  }
  const float c = A.scale * XA_LOG2E;
  const int qrow = (int)A.qs[1] * 2, qhead = (int)A.qs[2] * 2, grow = (int)A.gs[1] * 2, ghead = (int)A.gs[2] * 2;
  const int srow = wave * RPI + lane / NC, sc = (lane % NC) ^ xa_swz<RB>(srow);
  const unsigned dead = sc * 8 >= A.D ? XA_OOB : 0u;
  const float inv_lq = 1.f / (float)A.Lq;
  const int sg = STEP / A.Lq, sr = STEP - sg * A.Lq;              // STEP rows on: sg heads and sr rows, or a head more
  const unsigned qstep = (unsigned)(sr * qrow) + (unsigned)sg * (unsigned)qhead, gstep = (unsigned)(sr * grow) + (unsigned)sg * (unsigned)ghead;
  const unsigned qover = qstep + (unsigned)qhead - (unsigned)A.Lq * (unsigned)qrow, gover = gstep + (unsigned)ghead - (unsigned)A.Lq * (unsigned)grow;
  while (unit < end) {
    const long long flat = unit / per;                            // which 64 keys
    const int t0 = (int)(unit - flat * per);
    int t1 = end - unit < per - t0 ? t0 + (int)(end - unit) : per;
    const bool whole = t0 == 0 && t1 == per;
    unit += t1 - t0;
    int b, hk, tile;
    if (A.ragged) {
      int lo = 0, hi = A.B;                                       // the last entry that begins at `flat` or before it
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((long long)__builtin_amdgcn_readfirstlane(before[mid]) * A.Hkv <= flat) lo = mid; else hi = mid;
      }
      const int first = __builtin_amdgcn_readfirstlane(before[lo]), many = __builtin_amdgcn_readfirstlane(before[lo + 1]) - first;
      const int in = (int)(flat - (long long)first * A.Hkv);
      b = lo;
      hk = in / many;
      tile = in - hk * many;
    } else {
      const int head = (int)(flat / A.tiles);
      tile = (int)(flat - (long long)head * A.tiles);
      b = head / A.Hkv;
      hk = head - b * A.Hkv;
    }
    const long long head = (long long)b * A.Hkv + hk;
    const int key = tile * 64 + (wave & 1) * 32 + (lane & 31), nk = xa_keys(A, b);
    const bool counts = key < nk && (!A.mask || A.mask[(long long)b * A.ms + key]);
    const T* kp = (const T*)A.k + (long long)b * A.ks[0] + (long long)key * A.ks[1] + (long long)hk * A.ks[2];
    const T* vp = (const T*)A.v + (long long)b * A.vs[0] + (long long)key * A.vs[1] + (long long)hk * A.vs[2];
    u32x4 fk[KS], fv[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = s * 16 + h * 8;
      const bool ok = counts && d < A.D;
      fk[s] = ok ? *reinterpret_cast<const u32x4*>(kp + d) : u32x4{0, 0, 0, 0};
      fv[s] = ok ? *reinterpret_cast<const u32x4*>(vp + d) : u32x4{0, 0, 0, 0};
    }
    if (tile * 64 >= nk) t1 = t0;                                 // no key here counts: zeros
    const char* qp = (const char*)((const T*)A.q + (long long)b * A.qs[0] + (long long)hk * A.G * A.qs[2]);
    const char* gp = (const char*)((const T*)A.dout + (long long)b * A.gs[0] + (long long)hk * A.G * A.gs[2]);
    const __amdgpu_buffer_rsrc_t rq = xa_rsrc(qp), rg = xa_rsrc(gp);   // (host-checked: the heads of a group stay below 2^31 bytes)
    const __amdgpu_buffer_rsrc_t rl = xa_rsrc(A.lse2 + head * A.rows), rd = xa_rsrc(A.delta + head * A.rows);
    // where this lane's next row of Q and of dO lies: tiles are asked for in order, STEP rows an instruction
    int qi;
    const int g0 = fast_div(t0 * ROWS + srow, A.Lq, inv_lq, qi);
    unsigned oq = (unsigned)qi * (unsigned)qrow + (unsigned)g0 * (unsigned)qhead + (unsigned)(sc * 16);
    unsigned og = (unsigned)qi * (unsigned)grow + (unsigned)g0 * (unsigned)ghead + (unsigned)(sc * 16);
    auto issue = [&](int t, int buf) {
      char* st = smem + buf * STAGE;
      char* dst = st + wave * RPI * RB;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const unsigned bad = (srow < A.rows - t * ROWS - i * STEP ? 0u : XA_OOB) | dead;
        xa_dma16(rq, oq | bad, 0, dst + i * STEP * RB);
        xa_dma16(rg, og | bad, 0, dst + TILE + i * STEP * RB);
        qi += sr;
        const bool over = qi >= A.Lq;
        qi -= over ? A.Lq : 0;
        oq += over ? qover : qstep;
        og += over ? gover : gstep;
      }
      const int part = wave % RG, r = t * ROWS + part * 64 + lane;
      const unsigned off = r < A.rows ? (unsigned)r * 4u : XA_OOB;
      if (wave < RG) xa_dma4(rl, off, st + 2 * TILE + part * 256);
      else xa_dma4(rd, off, st + 2 * TILE + 4 * ROWS + part * 256);
    };
    const bool few = nk <= 64 * XA_FEW;
    float es = XaRange<T>::on ? 0x1p9f : 1.f;                     // (times the 2^15 of P)
    f32x16 dv[DT], dk[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) dv[d] = dk[d] = xa_zero();
    XaTr<DP> tr(smem + grp * 64 * RB, lane);
    auto rows = [&](auto few_) {
      int buf = 0;
      if (t0 < t1) issue(t0, 0);
      for (int t = t0; t < t1; ++t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + 1 < t1) issue(t + 1, buf ^ 1);
        const char* qt = smem + buf * STAGE + grp * 64 * RB;
        const char* gt = qt + TILE;
        const float* rowv = reinterpret_cast<const float*>(smem + buf * STAGE + 2 * TILE) + grp * 64;
        auto rows32 = [&](auto u_) {
          constexpr int u = decltype(u_)::value;
          f32x16 s, dp;                                             // (dP - Dl: the sums begin at -Dl)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 d4 = *reinterpret_cast<const f32x4*>(rowv + ROWS + 32 * u + 8 * q + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) dp[4 * q + i] = d4[i];
          }
          xa_scores<T, DP, KS>(qt, gt, 32 * u, lane, fk, fv, s, dp);
          float mx = 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(rowv + 32 * u + 8 * q + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 4 * q + i;
              s[r] = xa_exp2(__builtin_fmaf(s[r], c, l4[i]));
              dp[r] *= s[r];
              if constexpr (XaRange<T>::on) mx = fmaxf(mx, fabsf(dp[r]));
            }
          }
          if constexpr (XaRange<T>::on) {
            xa_fit<DT>(counts ? mx : 0.f, es, dk);                    // (a hidden key's column is dropped: any size)
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] *= es;
          }
          auto add = [&](auto kb_) {
            constexpr int kb = decltype(kb_)::value;
            u32x4 fg[DT], fq[DT];
            xa_tr_frags<DP, u * 32 + kb * 16, TILE>(tr, fg);
            const u32x4 fp = xa_as_b<T>(s, kb);
#pragma unroll
            for (int d = 0; d < DT; ++d) dv[d] = xa_mma<T>(fg[d], fp, dv[d]);
            if constexpr (decltype(few_)::value) {
              const u32x4 rest = xa_rest<T>(s, kb, fp);
#pragma unroll
              for (int d = 0; d < DT; ++d) dv[d] = xa_mma<T>(fg[d], rest, dv[d]);
            }
            xa_tr_frags<DP, u * 32 + kb * 16>(tr, fq);
            const u32x4 fs = xa_as_b<T>(dp, kb);
#pragma unroll
            for (int d = 0; d < DT; ++d) dk[d] = xa_mma<T>(fq[d], fs, dk[d]);
            if constexpr (decltype(few_)::value) {
              const u32x4 rest = xa_rest<T>(dp, kb, fs);
#pragma unroll
              for (int d = 0; d < DT; ++d) dk[d] = xa_mma<T>(fq[d], rest, dk[d]);
            }
          };
          add(XaInt<0>{}), add(XaInt<1>{});
        };
        rows32(XaInt<0>{}), rows32(XaInt<1>{});
        tr.move(buf ? -STAGE : STAGE);
        buf ^= 1;
      }
    };
    if (few) rows(XaInt<1>{});
    else rows(XaInt<0>{});
    // the other row groups' sums go to the first group's waves, added in order
    const float fk_ = A.scale * XaRange<T>::p_down / es, fv_ = XaRange<T>::p_down;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    f32x4* ex = reinterpret_cast<f32x4*>(smem) + (wave & 1) * EX + lane;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      dk[d] *= fk_;
      dv[d] *= fv_;
      if (grp) {
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          f32x4* to = ex + (grp - 1) * 2 * EX + (d * 4 + (r >> 2)) * 64;
          to[0] = f32x4{dk[d][r], dk[d][r + 1], dk[d][r + 2], dk[d][r + 3]};
          to[DT * 4 * 64] = f32x4{dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]};
        }
      }
    }
    __syncthreads();
    if (!grp && key < A.Lk) {
#pragma unroll
      for (int o = 0; o < RG - 1; ++o)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            const f32x4* from = ex + o * 2 * EX + (d * 4 + (r >> 2)) * 64;
            const f32x4 x = from[0], y = from[DT * 4 * 64];
#pragma unroll
            for (int i = 0; i < 4; ++i) { dk[d][r + i] += x[i]; dv[d][r + i] += y[i]; }
          }
      // (a hidden key's column was computed from zeros and is dropped, whatever it holds)
      if (!counts) {
#pragma unroll
        for (int d = 0; d < DT; ++d) dk[d] = dv[d] = xa_zero();
      }
      if (whole) {
        T* pk = (T*)A.dk + (long long)b * A.dks[0] + (long long)key * A.dks[1] + (long long)hk * A.dks[2];
        T* pv = (T*)A.dv + (long long)b * A.dvs[0] + (long long)key * A.dvs[1] + (long long)hk * A.dvs[2];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            const int ch = d * 32 + 2 * r + 4 * h;
            if (ch < A.D) {
              *reinterpret_cast<u32x2*>(pk + ch) = u32x2{xa_pack<T>(dk[d][r], dk[d][r + 1]), xa_pack<T>(dk[d][r + 2], dk[d][r + 3])};
              *reinterpret_cast<u32x2*>(pv + ch) = u32x2{xa_pack<T>(dv[d][r], dv[d][r + 1]), xa_pack<T>(dv[d][r + 2], dv[d][r + 3])};
            }
          }
      } else {                                                    // [share][rows' begin left out, or their end][dk, dv][64][D]
        float* pk = A.part + ((2ll * share + (t0 == 0)) * 128 + (key & 63)) * A.D;
        float* pv = pk + 64 * A.D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            const int ch = d * 32 + 2 * r + 4 * h;
            if (ch < A.D) {
              *reinterpret_cast<f32x4*>(pk + ch) = f32x4{dk[d][r], dk[d][r + 1], dk[d][r + 2], dk[d][r + 3]};
              *reinterpret_cast<f32x4*>(pv + ch) = f32x4{dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]};
            }
          }
      }
    }
    __syncthreads();                                              // (the exchange has been read: the stages are free)
  }
}

// adds the parts of 64 keys whose rows were dealt to several shares; dk or dv by blockIdx.y.  Where lengths are counted, also
// the zeros of the 64s without keys.
template <typename T>
__global__ __launch_bounds__(256) void xattn_parts_kernel(XaArgs A) {
  __shared__ int before[XA_RAGGED + 1];
  xa_count(A, before);
  const XaShares S(A, before);
  const int head = blockIdx.x / A.tiles, tile = blockIdx.x - head * A.tiles, b = head / A.Hkv, hk = head - b * A.Hkv;
  long long flat = blockIdx.x;
  bool none = false;
  if (A.ragged) {
    const int many = before[b + 1] - before[b];
    flat = (long long)before[b] * A.Hkv + (long long)hk * many + tile;
    none = tile >= many;
  }
  int s0 = 0, s1 = 0;
  if (!none) {
    s0 = S.of(flat * S.per);
    s1 = S.of(flat * S.per + S.per - 1);
    if (s0 == s1) return;                                         // (written whole)
  }
  const int chunks = A.D >> 3, which = blockIdx.y;
  T* out = (T*)(which ? A.dv : A.dk);
  const long long* st = which ? A.dvs : A.dks;
  for (int i = threadIdx.x; i < 64 * chunks; i += 256) {
    const int k = i / chunks, d = (i - k * chunks) * 8, key = tile * 64 + k;
    if (key >= A.Lk) break;
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
    if (!none) {
      const float* p = A.part + ((2ll * s0 + 1) * 128 + which * 64 + k) * A.D + d;
      x = *reinterpret_cast<const f32x4*>(p);
      y = *reinterpret_cast<const f32x4*>(p + 4);
      for (int s = s0 + 1; s <= s1; ++s) {
        p = A.part + (2ll * s * 128 + which * 64 + k) * A.D + d;
        x += *reinterpret_cast<const f32x4*>(p);
        y += *reinterpret_cast<const f32x4*>(p + 4);
      }
    }
    *reinterpret_cast<u32x4*>(out + (long long)b * st[0] + (long long)key * st[1] + (long long)hk * st[2] + d) =
        u32x4{xa_pack<T>(x[0], x[1]), xa_pack<T>(x[2], x[3]), xa_pack<T>(y[0], y[1]), xa_pack<T>(y[2], y[3])};
  }
}

// adds the shares of dq up, 8 channels per thread
template <typename T>
__global__ __launch_bounds__(256) void xattn_sum_kernel(XaArgs A) {
  const int chunks = A.D >> 3;
  const long long all = (long long)A.B * A.Hkv * A.rows, i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= all * chunks) return;
  const long long flat = i / chunks;
  const int d = (int)(i - flat * chunks) * 8;
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, e = a;
  for (int s = 0; s < A.nsplit; ++s) {
    const float* p = A.part + (s * all + flat) * A.D + d;
    a += *reinterpret_cast<const f32x4*>(p);
    e += *reinterpret_cast<const f32x4*>(p + 4);
  }
  const int head = (int)(flat / A.rows), row = (int)(flat - (long long)head * A.rows);
  const int b = head / A.Hkv, hk = head % A.Hkv, g = row / A.Lq, l = row - g * A.Lq;
  *reinterpret_cast<u32x4*>((T*)A.dq + b * A.dqs[0] + l * A.dqs[1] + (long long)(hk * A.G + g) * A.dqs[2] + d) =
      u32x4{xa_pack<T>(a[0], a[1]), xa_pack<T>(a[2], a[3]), xa_pack<T>(e[0], e[1]), xa_pack<T>(e[2], e[3])};
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
// dk, dv: shares (0: a block for each 64 keys).  Counted in row tiles a block walks one after the other, with `slots` blocks at
// a time: whole 64s cost ceil(64s / slots) times their rows; shares an even part, and adding their ends up is worth about
// three tiles more (7.8 us, at 2.8 us a tile).  With lengths, three quarters of the keys are expected to count.
struct XaBwdPlan { int qtiles, qsplit, ktiles, shares; long long rows_all; };
static XaBwdPlan xa_bwd_plan(const ried_xattn_t& d) {
  const long long rows = d.heads / d.groups * d.queries, heads = d.batch * d.groups;
  XaBwdPlan p;
  p.rows_all = heads * rows;
  auto split = [](long long blocks, long long want, long long most) {
    long long n = want / (blocks > 0 ? blocks : 1);
    if (n > most) n = most;
    if (n > 32) n = 32;
    return (int)(n < 1 ? 1 : n);
  };
  p.qtiles = ceil_div(rows, 128);
  p.qsplit = split(p.qtiles * heads, 512, d.keys / 256);
  p.ktiles = ceil_div(d.keys, 64);
  const long long slots = d.dim <= 64 ? 512 : 256, per = ceil_div(rows, 128), all = p.ktiles * heads, units = all * per;
  const long long dealt = (d.lengths ? units - units / 4 : units) / slots + 3, kept = ((d.lengths ? all - all / 4 : all) + slots - 1) / slots * per;
  const long long most = units / 2;
  p.shares = dealt < kept && most > 1 && (!d.lengths || d.batch <= XA_RAGGED) ? (int)(most < slots ? most : slots) : 0;
  return p;
}

extern "C" long long ried_xattn_bwd_scratch_floats(long long batch, long long queries, long long keys, int heads,
                                                   int groups, int dim) {
  if (batch <= 0 || queries <= 0 || heads <= 0 || groups <= 0 || heads % groups) return 0;
  ried_xattn_t d = {};
  d.batch = batch; d.queries = queries; d.keys = keys; d.heads = heads; d.groups = groups; d.dim = dim;
  const XaBwdPlan p = xa_bwd_plan(d);
  const int some = 0;
  d.lengths = &some;                                              // (a plan with lengths may deal where one without does not)
  const int shares = p.shares ? p.shares : xa_bwd_plan(d).shares;
  const long long a = p.qsplit > 1 ? p.qsplit * p.rows_all * dim : 0, b = 256ll * shares * dim;
  return 2 * ((p.rows_all + 3) / 4 * 4) + (a > b ? a : b);
}

template <typename T, int DP>
static int xa_bwd_launch(XaArgs A, const XaBwdPlan& p, hipStream_t stream) {
  constexpr int lq = 2 * 2 * 64 * XaTile<DP>::RB, lk = 2 * XaKv<DP>::STAGE;
  for (int i = 0; i < 2; ++i) {
    const hipError_t e = hipFuncSetAttribute(i ? (const void*)xattn_dkv_kernel<T, DP> : (const void*)xattn_dq_kernel<T, DP>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, i ? lk : lq);
    RIED_CHECK_ARG(e == hipSuccess, "ried_xattn_bwd: LDS: %s", hipGetErrorString(e));
  }
  const int heads = A.B * A.Hkv;
  A.tiles = p.qtiles;
  A.nsplit = p.qsplit;
  hipLaunchKernelGGL((xattn_dq_kernel<T, DP>), dim3((unsigned)(A.tiles * A.nsplit * heads)), dim3(256), lq, stream, A);
  if (A.nsplit > 1)
    hipLaunchKernelGGL((xattn_sum_kernel<T>), dim3(ceil_div(p.rows_all * (A.D >> 3), 256)), dim3(256), 0, stream, A);
  if (A.Lk == 0) return RIED_OK;
  A.tiles = p.ktiles;
  A.nsplit = p.shares;
  A.ragged = p.shares && A.lengths;
  hipLaunchKernelGGL((xattn_dkv_kernel<T, DP>), dim3((unsigned)(p.shares ? p.shares : A.tiles * heads)), dim3(64 * XaKv<DP>::NW), lk, stream, A);
  if (p.shares)
    hipLaunchKernelGGL((xattn_parts_kernel<T>), dim3((unsigned)(A.tiles * heads), 2), dim3(256), 0, stream, A);
  return RIED_OK;
}
template <typename T>
static int xa_bwd_dim(const XaArgs& A, const XaBwdPlan& p, hipStream_t stream) {
  return A.D <= 32 ? xa_bwd_launch<T, 32>(A, p, stream) : A.D <= 64 ? xa_bwd_launch<T, 64>(A, p, stream)
       : A.D <= 96 ? xa_bwd_launch<T, 96>(A, p, stream) : xa_bwd_launch<T, 128>(A, p, stream);
}

extern "C" int ried_xattn_bwd(const ried_xattn_t* desc, hipStream_t stream) {
  if (int e = xa_check(desc, "ried_xattn_bwd", true)) return e;
  const ried_xattn_t& d = *desc;
  if (d.batch == 0) return RIED_OK;
  RIED_CHECK_ARG(d.queries > 0, "ried_xattn_bwd: no queries (dk and dv are zeros: fill them)");
  RIED_CHECK_ARG(d.lse && d.scratch, "ried_xattn_bwd: lse and ried_xattn_bwd_scratch_floats() of scratch are needed");
  const long long G = d.heads / d.groups;
  RIED_CHECK_ARG(G * d.queries < (1ll << 29), "ried_xattn_bwd: sizes out of range");
  for (const long long* s : {d.q_stride, d.dout_stride})
    RIED_CHECK_ARG((d.queries * s[1] + G * s[2]) * 2 < (1ll << 31),
                   "ried_xattn_bwd: the heads of a group span over 2^31 bytes of q or dout: pass fewer queries");
  XaArgs A = xa_args(d);
  const XaBwdPlan p = xa_bwd_plan(d);
  RIED_CHECK_ARG((long long)p.qtiles * p.qsplit * A.B * A.Hkv < (1ll << 24) && (long long)p.ktiles * A.B * A.Hkv < (1ll << 23),
                 "ried_xattn_bwd: too many blocks");
  const long long pad = (p.rows_all + 3) / 4 * 4;
  A.lse2 = d.scratch;
  A.delta = d.scratch + pad;
  A.part = d.scratch + 2 * pad;
  const int e = d.type == RIED_T_BF16 ? xa_bwd_dim<bf16_t>(A, p, stream) : xa_bwd_dim<_Float16>(A, p, stream);
  if (e) return e;
  RIED_CHECK_LAUNCH("ried_xattn_bwd");
  return RIED_OK;
}
