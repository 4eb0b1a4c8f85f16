// Cross attention to an encoder's states, forward:  S = scale q k^T over the keys that count, P = softmax S, o = P v.
// A row without keys gives zeros (and a log-sum of -infinity).
//
// Heads that share a key head are folded into its rows (row = head in group * queries + query), so that a tile of keys
// and values serves them all.
#include "xattn.h"

// fp16 weights are held times 2^7 (with the 2^8 that a running maximum may be behind: up to 2^15), so that 2^-31 of the
// largest still counts beside it; bf16 has fp32's range
template <typename T> constexpr float xa_up = 0.f;
template <> constexpr float xa_up<_Float16> = 7.f;

// ---------------------------------------------------------------------------------------------------------------------
// Tiles: a wave owns 32 rows, a block of NW waves 32 NW; tiles of 64 keys go HBM -> LDS by DMA, one barrier per tile.
// S^T = K Q^T leaves a row's scores in one lane pair, so the softmax runs in registers, and P^T is the B operand of
// O^T += V^T P^T as it stands.  The running maximum is raised only when a score exceeds it by more than 2^8 (the
// sums hold that in fp32): rescaling is rare after the first tile.
//
// P enters the second product rounded to the type, its row sum is not.  With u half a step (bf16 2^-8), independent roundings move
// the result by at most u / sqrt(3) sqrt(sum P^2 v^2), beside its own rounding u / sqrt(3) of it.  Measured in bf16 on normal
// values, from one row over 77 keys to 4096 rows over 4096: 0.0019 to 0.0024 of the result's norm, where products in 32 bits
// leave 0.0016 to 0.0017.  What the rounding leaves over as a second operand would take that away for half as many products
// again in every tile.
//
// Measured, 2 x 4096 rows over 4096 keys, 16 heads of 128 channels, bf16 (275 GFLOP): 262 to 283 us by card, 970 to 1050
// TFLOP/s, where a matrix product of 8192 reaches 1320; the matrix pipes are busy 46 % of the cycles, LDS bank conflicts
// are none.  Nothing bounds it alone: with four waves (287 us) the products by themselves took 140 us, with the softmax 177,
// with the DMA 225, with the LDS reads 283 - two waves of a SIMD overlap one's products with the other's exponentials
// only in part.  4 x 4096 rows over 657 to 1500 keys, 4 key heads of 64 channels (18 GFLOP): 34.8 us.  Measured and left out:
// the next tile's scores under this tile's exponentials in one wave (305 us), a higher wave priority around the
// products (287), one stage for V, three blocks per CU (they spill at 128 channels), reading fragments ahead (all within
// 1 %).  With few blocks: four stages (16.4 against 13.8 us for 3 x 333 rows over 777 keys of 5 x 80), keys whole (23.4
// against 13.7 + 5.4 for the join).
// ---------------------------------------------------------------------------------------------------------------------
template <int DP, int NW> struct XaFwd { static constexpr int STAGES = NW == 8 ? 3 : 2, LDS = STAGES * 2 * 64 * XaTile<DP>::RB; };
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, 2) void xattn_fwd_kernel(XaArgs A) {
  constexpr int KS = XaTile<DP>::KS, DT = XaTile<DP>::DT, RB = XaTile<DP>::RB, NC = XaTile<DP>::NC, RPI = XaTile<DP>::RPI;
  constexpr int TILE = 64 * RB, NI = 64 / NW / RPI, NST = XaFwd<DP, NW>::STAGES;   // NI: DMA instructions per wave and operand
  extern __shared__ __align__(16) char smem[];                    // [NST][K tile, V tile]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  int inner, head;
  xa_block(A.tiles * A.nsplit, A.B * A.Hkv, inner, head);
  const int b = head / A.Hkv, hk = head % A.Hkv, tile = inner % A.tiles, split = inner / A.tiles;
  const int row = tile * (32 * NW) + wave * 32 + (lane & 31);
  const bool live = row < A.rows;
  const int g = live ? row / A.Lq : 0, qi = live ? row - g * A.Lq : 0;
  const T* qp = (const T*)A.q + (long long)b * A.qs[0] + (long long)qi * A.qs[1] + (long long)(hk * A.G + g) * A.qs[2];
  u32x4 fq[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = s * 16 + h * 8;
    fq[s] = live && d < A.D ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{0, 0, 0, 0};
  }
  const int nk = xa_keys(A, b), ntile = (nk + 63) >> 6, per = (ntile + A.nsplit - 1) / A.nsplit;
  const int t0 = split * per, t1 = t0 + per < ntile ? t0 + per : ntile;
  const char* kp = (const char*)((const T*)A.k + (long long)b * A.ks[0] + (long long)hk * A.ks[2]);
  const char* vp = (const char*)((const T*)A.v + (long long)b * A.vs[0] + (long long)hk * A.vs[2]);
  const unsigned char* mp = A.mask ? A.mask + (long long)b * A.ms : nullptr;
  const int krow = (int)A.ks[1] * 2, vrow = (int)A.vs[1] * 2;    // bytes (host-checked: 64 rows stay below 2^31)
  const int srow = wave * RPI + lane / NC, sc = (lane % NC) ^ xa_swz<RB>(srow);
  const unsigned dead = sc * 8 >= A.D ? XA_OOB : 0u;
  const unsigned koff = (unsigned)(srow * krow + sc * 16) | dead, voff = (unsigned)(srow * vrow + sc * 16) | dead;
  auto issue = [&](int t, u64 w, int buf) {
    const __amdgpu_buffer_rsrc_t rk = xa_rsrc(kp + (long long)t * 64 * krow), rv = xa_rsrc(vp + (long long)t * 64 * vrow);
    char* dst = smem + buf * 2 * TILE + wave * RPI * RB;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const unsigned bad = (w >> (srow + i * NW * RPI)) & 1 ? 0u : XA_OOB;
      xa_dma16(rk, koff | bad, i * NW * RPI * krow, dst + i * NW * RPI * RB);
      xa_dma16(rv, voff | bad, i * NW * RPI * vrow, dst + TILE + i * NW * RPI * RB);
    }
  };
  auto mask_byte = [&](int t) -> int {
    const int key = t * 64 + lane;
    return mp && key < nk ? mp[key] : 0;
  };
  const float c = A.scale * XA_LOG2E;
  float m = -INFINITY, mc = 0.f, sum = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = xa_zero();
  XaTr<DP> tr(smem + TILE, lane);
  // Tiles are asked for NST - 1 ahead; past the end the DMA writes zeros, so that the counted wait holds.
  u64 w[NST] = {};
  int byte = 0, buf = 0;
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) {
    w[i] = t0 + i < t1 ? xa_word(nk - (t0 + i) * 64, mp != nullptr, mask_byte(t0 + i)) : 0;
    if (t0 < t1) issue(t0 + i < t1 ? t0 + i : t0, w[i], i);
  }
  if (t0 < t1) byte = mask_byte(t0 + NST - 1);
  for (int t = t0; t < t1; ++t) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 2) * 2 * NI) : "memory");
    __builtin_amdgcn_s_barrier();                                 // tile t has landed; everyone is done with the tile before it
    asm volatile("" ::: "memory");
    {
      const int n = t + NST - 1;
      w[NST - 1] = n < t1 ? xa_word(nk - n * 64, mp != nullptr, byte) : 0;
      byte = mask_byte(n + 1);
      issue(n < t1 ? n : t0, w[NST - 1], buf == 0 ? NST - 1 : buf - 1);
    }
    {
      const char* kt = smem + buf * 2 * TILE;
      f32x16 s[2] = {xa_zero(), xa_zero()};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] = xa_mma<T>(xa_frag<DP>(kt, 32 * u, ks, lane), fq[ks], s[u]);
      if (w[0] != ~0ull) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const unsigned bits = (unsigned)(w[0] >> (32 * u)) >> (4 * h);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = (bits >> (8 * (r >> 2) + (r & 3))) & 1 ? s[u][r] : -INFINITY;
        }
      }
      float mx = s[0][0];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[u][r]);
      if (__any((mx - m) * c > 8.f || (m == -INFINITY && mx > m))) {
        float lo, hi;
        xa_halves(mx, lo, hi);
        const float mn = fmaxf(m, fmaxf(lo, hi));
        const float nc = mn == -INFINITY ? 0.f : mn * c - xa_up<T>;
        const float a = xa_exp2((m == -INFINITY ? -INFINITY : mc) - nc);
        m = mn;
        mc = nc;
        sum *= a;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= a;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[u][r] = xa_exp2(__builtin_fmaf(s[u][r], c, -mc));
          sum += s[u][r];
        }
      auto add = [&](auto kb_) {
        constexpr int kb = decltype(kb_)::value;
        u32x4 fv[DT];
        xa_tr_frags<DP, kb * 16>(tr, fv);
        const u32x4 p = xa_as_b<T>(s[kb >> 1], kb & 1);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = xa_mma<T>(fv[d], p, acc[d]);
      };
      add(XaInt<0>{}), add(XaInt<1>{}), add(XaInt<2>{}), add(XaInt<3>{});
    }
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) w[i] = w[i + 1];
    tr.move(buf == NST - 1 ? -(NST - 1) * 2 * TILE : 2 * TILE);
    buf = buf == NST - 1 ? 0 : buf + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                // no DMA may outlive the block
  float lo, hi;
  xa_halves(sum, lo, hi);
  const float total = lo + hi;
  // (zero only for a row without keys: a row's largest weight is at least 1, or 2^7.  NaN goes on to the result.)
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const float lse = total == 0.f ? -INFINITY : (mc + __log2f(total)) * XA_LN2;
  if (!live) return;
  const long long flat = (long long)head * A.rows + row;
  if (A.nsplit == 1) {
    if (h == 0 && A.lse) A.lse[flat] = lse;
    T* op = (T*)A.out + (long long)b * A.os[0] + (long long)qi * A.os[1] + (long long)(hk * A.G + g) * A.os[2];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int ch = d * 32 + 2 * r + 4 * h;
        if (ch < A.D)
          *reinterpret_cast<u32x2*>(op + ch) = u32x2{xa_pack<T>(acc[d][r] * inv, acc[d][r + 1] * inv),
                                                     xa_pack<T>(acc[d][r + 2] * inv, acc[d][r + 3] * inv)};
      }
  } else {
    const long long at = (long long)split * A.B * A.Hkv * A.rows + flat;
    if (h == 0) A.part_lse[at] = lse;
    float* op = A.part + at * A.D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int ch = d * 32 + 2 * r + 4 * h;
        if (ch < A.D)
          *reinterpret_cast<f32x4*>(op + ch) = f32x4{acc[d][r] * inv, acc[d][r + 1] * inv, acc[d][r + 2] * inv, acc[d][r + 3] * inv};
      }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Few rows (up to 32 per key head: single tokens): the four waves of a block take turns at tiles of 32 keys of the block's
// share of the keys, each with two DMA stages of its own (no barrier in the loop), and are joined through LDS.  Bound by the
// keys' and values' bytes: 16 x 1 token over 1216 to 4096 keys, 8 key heads for 32 of 128 channels, 174 MB: 40.7 us
// (4.3 TB/s) + 4.9 for the join.  (Shares for 512 or 1024 blocks instead of 256: 44.1 and 48.4 us in all against 44.9.)
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(256, 1) void xattn_token_kernel(XaArgs A) {
  constexpr int KS = XaTile<DP>::KS, DT = XaTile<DP>::DT, RB = XaTile<DP>::RB, NC = XaTile<DP>::NC, RPI = XaTile<DP>::RPI;
  constexpr int TILE = 32 * RB, NI = 32 / RPI, PO = DP + 4;       // PO: row pitch (floats) of the exchange
  static_assert(4 * (32 * PO + 64) * 4 <= 4 * 2 * 2 * TILE, "the exchange reuses the stages");
  extern __shared__ __align__(16) char smem[];                    // [4 waves][2 stages][K tile, V tile]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  int split, head;
  xa_block(A.nsplit, A.B * A.Hkv, split, head);
  const int b = head / A.Hkv, hk = head % A.Hkv, row = lane & 31;
  const bool live = row < A.rows;
  const int g = live ? row / A.Lq : 0, qi = live ? row - g * A.Lq : 0;
  const T* qp = (const T*)A.q + (long long)b * A.qs[0] + (long long)qi * A.qs[1] + (long long)(hk * A.G + g) * A.qs[2];
  u32x4 fq[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = s * 16 + h * 8;
    fq[s] = live && d < A.D ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{0, 0, 0, 0};
  }
  const int nk = xa_keys(A, b), ntile = (nk + 31) >> 5, per = (ntile + A.nsplit - 1) / A.nsplit;
  const int t0 = split * per + wave, t1 = split * per + per < ntile ? split * per + per : ntile;
  const char* kp = (const char*)((const T*)A.k + (long long)b * A.ks[0] + (long long)hk * A.ks[2]);
  const char* vp = (const char*)((const T*)A.v + (long long)b * A.vs[0] + (long long)hk * A.vs[2]);
  const unsigned char* mp = A.mask ? A.mask + (long long)b * A.ms : nullptr;
  const int krow = (int)A.ks[1] * 2, vrow = (int)A.vs[1] * 2;
  const int srow = lane / NC;
  char* const base = smem + wave * 4 * TILE;
  XaTr<DP> tr(base + TILE, lane);
  // (a wave's DMA instruction i fills rows i * RPI ..; with RPI = 4 the swizzle of odd i differs)
  auto issue = [&](int t, unsigned w, int buf) {
    const __amdgpu_buffer_rsrc_t rk = xa_rsrc(kp + (long long)t * 32 * krow), rv = xa_rsrc(vp + (long long)t * 32 * vrow);
    char* dst = base + buf * 2 * TILE;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = srow + i * RPI, sc = (lane % NC) ^ xa_swz<RB>(r);
      const unsigned bad = ((w >> r) & 1) && sc * 8 < A.D ? 0u : XA_OOB;
      xa_dma16(rk, (unsigned)(srow * krow + sc * 16) | bad, i * RPI * krow, dst + i * RPI * RB);
      xa_dma16(rv, (unsigned)(srow * vrow + sc * 16) | bad, i * RPI * vrow, dst + TILE + i * RPI * RB);
    }
  };
  auto mask_byte = [&](int t) -> int {
    const int key = t * 32 + (lane & 31);
    return mp && key < nk ? mp[key] : 0;
  };
  auto word = [&](int t, int byte) -> unsigned {
    return t < t1 ? (unsigned)xa_word(nk - t * 32, mp != nullptr, byte) : 0u;
  };
  const float c = A.scale * XA_LOG2E;
  float m = -INFINITY, mc = 0.f, sum = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = xa_zero();
  if (t0 < t1) {
    int byte = mask_byte(t0), byte1 = mask_byte(t0 + 4);
    unsigned w = word(t0, byte), w1 = word(t0 + 4, byte1);
    issue(t0, w, 0);
    byte = mask_byte(t0 + 8);
    issue(t0 + 4 < t1 ? t0 + 4 : t0, w1, 1);                      // (past the end: zeros, so that the count holds)
    int buf = 0;
    for (int t = t0; t < t1; t += 4) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NI) : "memory");
      const char* kt = base + buf * 2 * TILE;
      f32x16 s = xa_zero();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = xa_mma<T>(xa_frag<DP>(kt, 0, ks, lane), fq[ks], s);
      if ((w & 0xffffffffu) != 0xffffffffu) {
        const unsigned bits = w >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (bits >> (8 * (r >> 2) + (r & 3))) & 1 ? s[r] : -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
      if (__any((mx - m) * c > 8.f || (m == -INFINITY && mx > m))) {
        float lo, hi;
        xa_halves(mx, lo, hi);
        const float mn = fmaxf(m, fmaxf(lo, hi));
        const float nc = mn == -INFINITY ? 0.f : mn * c - xa_up<T>;
        const float a = xa_exp2((m == -INFINITY ? -INFINITY : mc) - nc);
        m = mn;
        mc = nc;
        sum *= a;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= a;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = xa_exp2(__builtin_fmaf(s[r], c, -mc));
        sum += s[r];
      }
      auto add = [&](auto kb_) {
        constexpr int kb = decltype(kb_)::value;
        u32x4 fv[DT];
        xa_tr_frags<DP, kb * 16>(tr, fv);
        const u32x4 p = xa_as_b<T>(s, kb);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = xa_mma<T>(fv[d], p, acc[d]);
      };
      add(XaInt<0>{}), add(XaInt<1>{});
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // this stage has been read
      const unsigned w2 = word(t + 8, byte);
      byte = mask_byte(t + 12);
      issue(t + 8 < t1 ? t + 8 : t0, w2, buf);
      w = w1;
      w1 = w2;
      tr.move(buf ? -2 * TILE : 2 * TILE);
      buf ^= 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                // no DMA may land in the exchange
  __syncthreads();
  float* ex = reinterpret_cast<float*>(smem) + wave * (32 * PO + 64);
  {
    float lo, hi;
    xa_halves(sum, lo, hi);
    if (h == 0) {
      ex[32 * PO + row] = m == -INFINITY ? -INFINITY : mc;
      ex[32 * PO + 32 + row] = lo + hi;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<f32x4*>(ex + row * PO + d * 32 + 2 * r + 4 * h) = f32x4{acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]};
  }
  __syncthreads();
  const float* e0 = reinterpret_cast<const float*>(smem);
  for (int i = tid; i < A.rows * (DP / 4); i += 256) {
    const int r = i / (DP / 4), d = (i % (DP / 4)) * 4;
    float top = -INFINITY, tot = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float mk = e0[k * (32 * PO + 64) + 32 * PO + r];
      top = mk > top || mk != mk ? mk : top;
    }
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* e = e0 + k * (32 * PO + 64);
      const float mk = e[32 * PO + r], f = mk == -INFINITY ? 0.f : xa_exp2(mk - top);
      tot += e[32 * PO + 32 + r] * f;
      o += *reinterpret_cast<const f32x4*>(e + r * PO + d) * f;
    }
    const float inv = tot == 0.f ? 0.f : 1.f / tot;
    const float lse = tot == 0.f ? -INFINITY : (top + __log2f(tot)) * XA_LN2;
    const long long flat = (long long)head * A.rows + r;
    o *= inv;
    if (A.nsplit == 1) {
      const int gg = r / A.Lq, qq = r - gg * A.Lq;
      if (d == 0 && A.lse) A.lse[flat] = lse;
      if (d < A.D)
        *reinterpret_cast<u32x2*>((T*)A.out + (long long)b * A.os[0] + (long long)qq * A.os[1] +
                                  (long long)(hk * A.G + gg) * A.os[2] + d) = u32x2{xa_pack<T>(o[0], o[1]), xa_pack<T>(o[2], o[3])};
    } else {
      const long long at = (long long)split * A.B * A.Hkv * A.rows + flat;
      if (d == 0) A.part_lse[at] = lse;
      if (d < A.D) *reinterpret_cast<f32x4*>(A.part + at * A.D + d) = o;
    }
  }
}

// joins the shares of the keys: a wave per row (a thread per 8 channels of a row took 26 us for 64 shares of one row, this
// 4.7).  The shares' weights are formed by one lane each (up to 64 shares); 16 lanes
// by 8 channels take every fourth share each, so a row's loads are in flight together, and the four sums are added.
template <typename T>
__global__ __launch_bounds__(256) void xattn_join_kernel(XaArgs A) {
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const long long all = (long long)A.B * A.Hkv * A.rows, flat = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (flat >= all) return;
  const float l = lane < A.nsplit ? A.part_lse[lane * all + flat] : -INFINITY;
  float top = l;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float x = __shfl_xor(top, o, 64);
    top = x > top || x != x ? x : top;                            // (NaN wins)
  }
  const float w = l == -INFINITY ? 0.f : xa_exp2((l - top) * XA_LOG2E);
  const float tot = wave_sum(w);
  float o[8] = {};
  const bool has = c * 8 < A.D;
  for (int s0 = 0; s0 < A.nsplit; s0 += 16) {                     // (the same trips for every lane: the weights change lanes)
    f32x4 x[4], y[4];
    float f[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + 4 * u + q;
      f[u] = __shfl(w, s & 63, 64);
      x[u] = y[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (has && s < A.nsplit && f[u] != 0.f) {                   // (a share without keys wrote zeros)
        const float* p = A.part + (s * all + flat) * A.D + c * 8;
        x[u] = *reinterpret_cast<const f32x4*>(p);
        y[u] = *reinterpret_cast<const f32x4*>(p + 4);
      } else {
        f[u] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) { o[k] += x[u][k] * f[u]; o[4 + k] += y[u][k] * f[u]; }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = rows_sum(o[k]);
  const float inv = tot == 0.f ? 0.f : 1.f / tot;
  const int head = (int)(flat / A.rows), row = (int)(flat - (long long)head * A.rows);
  const int b = head / A.Hkv, hk = head % A.Hkv, g = row / A.Lq, qi = row - g * A.Lq;
  if (lane == 0 && A.lse) A.lse[flat] = tot == 0.f ? -INFINITY : top + __logf(tot);
  if (q == 0 && has) {
    T* op = (T*)A.out + (long long)b * A.os[0] + (long long)qi * A.os[1] + (long long)(hk * A.G + g) * A.os[2] + c * 8;
    *reinterpret_cast<u32x4*>(op) = u32x4{xa_pack<T>(o[0] * inv, o[1] * inv), xa_pack<T>(o[2] * inv, o[3] * inv),
                                          xa_pack<T>(o[4] * inv, o[5] * inv), xa_pack<T>(o[6] * inv, o[7] * inv)};
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
struct XaSplit { int tiles, nsplit, nw; };
// Waves a block, row tiles and shares of the keys.  Where blocks of eight waves (256 rows) give every CU one, they are taken -
// half the DMA a row - and the keys stay whole; with ragged lengths only where there are several per CU, because blocks
// then differ (4 x 4096 rows over 657 to 1500 keys: 35 us with four waves, 39 with eight).  Otherwise four waves, and the
// keys are shared out until there are 512 blocks (256 for single tokens at D > 64, one per CU), a share keeping at least
// four tiles per wave that reads it.  The shares do not depend on `lengths`: the scratch size has to be known without.
static XaSplit xa_fwd_split(const ried_xattn_t& d) {
  const long long rows = d.heads / d.groups * d.queries, heads = d.batch * d.groups, wide = ceil_div(rows, 256) * heads;
  XaSplit s;
  s.nw = rows > 128 && wide >= (d.lengths ? 1024 : 256) ? 8 : 4;
  s.tiles = rows <= 32 ? 1 : ceil_div(rows, 32 * s.nw);
  s.nsplit = 1;
  if (rows > 128 && wide >= 256) return s;
  const long long blocks = s.tiles * heads, want = rows <= 32 && d.dim > 64 ? 256 : 512, most = rows <= 32 ? d.keys / 512 : d.keys / 256;
  long long n = want / (blocks > 0 ? blocks : 1);
  if (n > most) n = most;
  if (n > 64) n = 64;
  s.nsplit = n < 1 ? 1 : (int)n;
  return s;
}

int xa_check(const ried_xattn_t* d, const char* name, bool bwd) {
  RIED_CHECK_ARG(d, "%s: null descriptor", name);
  RIED_CHECK_ARG(d->type == RIED_T_BF16 || d->type == RIED_T_F16, "%s: types are 1 bf16, 2 fp16", name);
  RIED_CHECK_ARG(d->batch >= 0 && d->queries >= 0 && d->keys >= 0 && d->heads > 0 && d->groups > 0 && d->heads % d->groups == 0,
                 "%s: bad sizes (batch %lld, queries %lld, keys %lld, heads %lld over %lld key heads)", name, d->batch,
                 d->queries, d->keys, d->heads, d->groups);
  RIED_CHECK_ARG(d->dim >= 8 && d->dim <= 128 && d->dim % 8 == 0, "%s: head dimension %lld is not a multiple of 8 up to 128", name, d->dim);
  RIED_CHECK_ARG(d->keys <= (1ll << 30) && d->queries <= (1ll << 30) && d->batch <= (1ll << 20) && d->heads <= (1ll << 20) &&
                 d->heads / d->groups * d->queries <= (1ll << 30) && d->batch * d->groups <= (1ll << 24),
                 "%s: sizes out of range", name);
  // (below, the kernels' factor would be zero in 32 bits, and zero times a hidden key's -infinity is not a number)
  RIED_CHECK_ARG(d->scale > 1e-37 && d->scale < 1e30, "%s: the scale is a positive number between 1e-37 and 1e30", name);
  if (d->batch == 0 || d->queries == 0) return RIED_OK;
  struct View { const void* p; const long long* s; const char* n; bool need; } views[] = {
      {d->q, d->q_stride, "q", true}, {d->k, d->k_stride, "k", d->keys > 0}, {d->v, d->v_stride, "v", d->keys > 0},
      {d->o, d->o_stride, "o", true}, {d->dout, d->dout_stride, "dout", bwd}, {d->dq, d->dq_stride, "dq", bwd},
      {d->dk, d->dk_stride, "dk", bwd && d->keys > 0}, {d->dv, d->dv_stride, "dv", bwd && d->keys > 0}};
  for (const View& v : views) {
    if (!v.need) continue;
    RIED_CHECK_ARG(v.p && ((uintptr_t)v.p & 15) == 0, "%s: %s is null or not 16-byte aligned", name, v.n);
    for (int i = 0; i < 3; ++i)
      RIED_CHECK_ARG(v.s[i] >= 0 && v.s[i] % 8 == 0, "%s: strides of %s are multiples of 8 elements", name, v.n);
    RIED_CHECK_ARG(v.s[1] <= (1 << 23), "%s: token stride of %s is over 2^23 elements", name, v.n);
  }
  return RIED_OK;
}

XaArgs xa_args(const ried_xattn_t& d) {
  XaArgs A = {};
  A.q = d.q; A.k = d.k; A.v = d.v; A.o = d.o; A.out = d.o; A.dout = d.dout; A.dq = d.dq; A.dk = d.dk; A.dv = d.dv;
  A.lse = d.lse; A.lengths = d.lengths; A.mask = d.key_mask; A.ms = d.mask_stride;
  for (int i = 0; i < 3; ++i) {
    A.qs[i] = d.q_stride[i]; A.ks[i] = d.k_stride[i]; A.vs[i] = d.v_stride[i]; A.os[i] = d.o_stride[i];
    A.gs[i] = d.dout_stride[i]; A.dqs[i] = d.dq_stride[i]; A.dks[i] = d.dk_stride[i]; A.dvs[i] = d.dv_stride[i];
  }
  A.B = (int)d.batch; A.Lq = (int)d.queries; A.Lk = (int)d.keys; A.Hkv = (int)d.groups; A.G = (int)(d.heads / d.groups);
  A.D = (int)d.dim; A.rows = A.G * A.Lq; A.scale = (float)d.scale;
  return A;
}

extern "C" long long ried_xattn_fwd_scratch_floats(long long batch, long long queries, long long keys, int heads,
                                                   int groups, int dim) {
  if (batch <= 0 || queries <= 0 || heads <= 0 || groups <= 0 || heads % groups) return 0;
  ried_xattn_t d = {};
  d.batch = batch; d.queries = queries; d.keys = keys; d.heads = heads; d.groups = groups; d.dim = dim;
  const XaSplit s = xa_fwd_split(d);
  return s.nsplit == 1 ? 0 : s.nsplit * batch * heads * queries * (dim + 1);
}

template <typename K>
static int xa_lds(K kernel, int bytes, const char* name) {
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  RIED_CHECK_ARG(e == hipSuccess, "%s: %d bytes of LDS: %s", name, bytes, hipGetErrorString(e));
  return RIED_OK;
}

template <typename T, int DP>
static int xa_fwd_launch(const XaArgs& A, hipStream_t stream) {
  const unsigned grid = (unsigned)(A.tiles * A.nsplit * A.B * A.Hkv);
  if (A.rows <= 32) {
    constexpr int lds = 4 * 2 * 2 * 32 * XaTile<DP>::RB;
    if (int e = xa_lds(xattn_token_kernel<T, DP>, lds, "ried_xattn_fwd")) return e;
    hipLaunchKernelGGL((xattn_token_kernel<T, DP>), dim3(grid), dim3(256), lds, stream, A);
  } else {
    constexpr int lds4 = XaFwd<DP, 4>::LDS, lds8 = XaFwd<DP, 8>::LDS;
    if (A.nw == 8) {
      if (int e = xa_lds(xattn_fwd_kernel<T, DP, 8>, lds8, "ried_xattn_fwd")) return e;
      hipLaunchKernelGGL((xattn_fwd_kernel<T, DP, 8>), dim3(grid), dim3(512), lds8, stream, A);
    } else {
      if (int e = xa_lds(xattn_fwd_kernel<T, DP, 4>, lds4, "ried_xattn_fwd")) return e;
      hipLaunchKernelGGL((xattn_fwd_kernel<T, DP, 4>), dim3(grid), dim3(256), lds4, stream, A);
    }
  }
  if (A.nsplit > 1)
    hipLaunchKernelGGL((xattn_join_kernel<T>), dim3(ceil_div((long long)A.B * A.Hkv * A.rows, 4)), dim3(256), 0, stream, A);
  return RIED_OK;
}
template <typename T>
static int xa_fwd_dim(const XaArgs& A, hipStream_t stream) {
  return A.D <= 32 ? xa_fwd_launch<T, 32>(A, stream) : A.D <= 64 ? xa_fwd_launch<T, 64>(A, stream)
       : A.D <= 96 ? xa_fwd_launch<T, 96>(A, stream) : xa_fwd_launch<T, 128>(A, stream);
}

extern "C" int ried_xattn_fwd(const ried_xattn_t* desc, hipStream_t stream) {
  if (int e = xa_check(desc, "ried_xattn_fwd", false)) return e;
  const ried_xattn_t& d = *desc;
  if (d.batch == 0 || d.queries == 0) return RIED_OK;
  XaArgs A = xa_args(d);
  const XaSplit s = xa_fwd_split(d);
  A.tiles = s.tiles;
  A.nsplit = s.nsplit;
  A.nw = s.nw;
  RIED_CHECK_ARG((long long)A.tiles * A.nsplit * A.B * A.Hkv * 64 * A.nw < (1ll << 32), "ried_xattn_fwd: too many blocks");
  if (A.nsplit > 1) {
    RIED_CHECK_ARG(d.scratch, "ried_xattn_fwd: this call needs ried_xattn_fwd_scratch_floats() of scratch");
    A.part = d.scratch;
    A.part_lse = d.scratch + (long long)A.nsplit * A.B * A.Hkv * A.rows * A.D;
  }
  const int e = d.type == RIED_T_BF16 ? xa_fwd_dim<bf16_t>(A, stream) : xa_fwd_dim<_Float16>(A, stream);
  if (e) return e;
  RIED_CHECK_LAUNCH("ried_xattn_fwd");
  return RIED_OK;
}
