// Shared pieces of the cross-attention kernels (forward, single-token forward, backward).
//
// MFMA v_mfma_f32_32x32x16, D[i][j] += sum_k A[i][k] B[k][j], 64 lanes, h = lane >> 5, l = lane & 31:
//   A operand  lane supplies A[i = l][k = 8h .. 8h+7]
//   B operand  lane supplies B[k = 8h .. 8h+7][j = l]
//   D          lane holds    D[i = 8 (r / 4) + 4h + r % 4][j = l], r = 0..15
// The order of k inside a 16-slice is free as long as both operands agree: a result is fed back as a B operand
// (contraction over its i index) by packing r = 0..7 and r = 8..15 as they stand, which is k = {4h.., 8 + 4h..}; the
// matching A operand comes out of LDS through the transposing read with its k rows addressed in that order.
//
// An LDS tile holds 64 rows (keys, or query rows) of 128 or 256 bytes; 16-byte chunk c of row r is stored in slot
// c ^ swz(r).  The LDS serves 256 bytes a cycle: 16 lanes of a row-wise 16-byte read, whose 16 rows put a chunk into 16
// different places of the 256 bytes, or 32 lanes of a transposing 8-byte read, which takes 64 bytes of 4 rows.  (Measured:
// 4 and 2 cycles an instruction without conflicts; a swizzle over 8 places cost the former 4 more.)  Tiles are filled by LDS
// DMA: its destination is lane-linear, so the swizzle is applied to the chunk a lane fetches; rows and chunks that do not
// exist (past the end, hidden keys, channels past D) use an offset outside the descriptor and arrive as zeros - whatever
// a hidden key holds never reaches a product.
#pragma once
#include "tokens.h"
#include "../../include/ried_gan.h"

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 pk_f16x2;
typedef __attribute__((address_space(3))) s16x4 xa_lds_s16x4;
typedef unsigned long long u64;

template <int N> struct XaInt { static constexpr int value = N; };
#define XA_OOB 0x80000000u
#define XA_LOG2E 1.44269504088896340736f
#define XA_LN2 0.69314718055994530942f

template <typename T> __device__ __forceinline__ f32x16 xa_mma(u32x4 a, u32x4 b, f32x16 c);
template <> __device__ __forceinline__ f32x16 xa_mma<bf16_t>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 xa_mma<_Float16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <typename T> __device__ __forceinline__ unsigned xa_pack(float lo, float hi);
template <> __device__ __forceinline__ unsigned xa_pack<bf16_t>(float lo, float hi) { return pack2bf(lo, hi); }
template <> __device__ __forceinline__ unsigned xa_pack<_Float16>(float lo, float hi) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(pk_f32x2{lo, hi}, pk_f16x2));
}
template <typename T> __device__ __forceinline__ void xa_unpack(u32x4 u, float (&f)[8]) {
  const TokVec<T, 8> v = __builtin_bit_cast(TokVec<T, 8>, u);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = TokType<T>::up(v.e[i]);
}
// rows 16 * which .. of a result, as the B operand of a product over its rows
template <typename T> __device__ __forceinline__ u32x4 xa_as_b(const f32x16& s, int which) {
  const int o = 8 * which;
  return u32x4{xa_pack<T>(s[o], s[o + 1]), xa_pack<T>(s[o + 2], s[o + 3]), xa_pack<T>(s[o + 4], s[o + 5]), xa_pack<T>(s[o + 6], s[o + 7])};
}
__device__ __forceinline__ f32x16 xa_zero() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

template <int RB> __device__ __forceinline__ int xa_swz(int r) {
  return RB == 256 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// (lo, hi): this lane's value and that of lane ^ 32, in lane order
__device__ __forceinline__ void xa_halves(float v, float& lo, float& hi) {
  lo = v;
  hi = v;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));   // lo lanes 32..63 <-> hi lanes 0..31
}

__device__ __forceinline__ void xa_dma16(__amdgpu_buffer_rsrc_t rsrc, unsigned off, int soff, char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, (int)off, soff, 0, 0);
}
__device__ __forceinline__ void xa_dma4(__amdgpu_buffer_rsrc_t rsrc, unsigned off, char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 4, (int)off, 0, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t xa_rsrc(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00020000);
}
__device__ __forceinline__ float xa_exp2(float v) { return __builtin_amdgcn_exp2f(v); }

// Geometry of a tile for head dimensions up to DP
template <int DP> struct XaTile {
  static constexpr int KS = DP / 16, DT = DP / 32, RB = DP <= 64 ? 128 : 256, NC = RB / 16, RPI = 64 / NC;
};

// Fragment of 32 rows from `rowbase` of a tile, channels 16 ks .. + 15, as an A (or B) operand over the channels
template <int DP>
__device__ __forceinline__ u32x4 xa_frag(const char* tile, int rowbase, int ks, int lane) {
  constexpr int RB = XaTile<DP>::RB;
  const int r = lane & 31, c = (2 * ks + (lane >> 5)) ^ xa_swz<RB>(r);
  return *reinterpret_cast<const u32x4*>(tile + (rowbase + r) * RB + c * 16);
}
// Fragments of channels 32 dt .. + 31 (the operand's rows) for all dt, contraction over the 16 tile rows from ROW (paired
// order).  Written in assembly, its wait included: the compiler cannot tell the transposing read from the DMA stage that
// is being filled and would wait for that first, which puts a memory round trip into every tile.
template <int DP> struct XaTr {
  unsigned at[2][XaTile<DP>::DT];                                 // this lane's LDS addresses in a tile: rows k0, k0 + 8
  __device__ __forceinline__ XaTr(const char* tile, int lane) {
    constexpr int RB = XaTile<DP>::RB;
    const int h = lane >> 5, rg = (lane >> 4) & 1, q = (lane >> 2) & 3, p = lane & 3, k0 = 4 * h + q;
    static_assert(RB == 256 || XaTile<DP>::DT <= 2, "chunks of a row");
    const unsigned t = (unsigned)(unsigned long long)(__attribute__((address_space(3))) const char*)tile + k0 * RB + (p & 1) * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < XaTile<DP>::DT; ++d) at[i][d] = t + 16 * ((d * 4 + rg * 2 + (p >> 1)) ^ xa_swz<RB>(k0 + 8 * i));
  }
  __device__ __forceinline__ void move(int bytes) {               // to another tile
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < XaTile<DP>::DT; ++d) at[i][d] += bytes;
  }
};
template <int DP, int ROW, int MORE = 0>                           // MORE: bytes from the tile that `a` points at
__device__ __forceinline__ void xa_tr_frags(const XaTr<DP>& a, u32x4 (&f)[XaTile<DP>::DT]) {
  constexpr int RB = XaTile<DP>::RB, DT = XaTile<DP>::DT, OFF = ROW * RB + MORE;
  static_assert(OFF + 8 * RB < 65536, "LDS instruction offset");
  u32x2 lo[DT], hi[DT];
  if constexpr (DT == 1) {
    asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%4\n\t"
                 "ds_read_b64_tr_b16 %1, %3 offset:%5\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0])
                 : "v"(a.at[0][0]), "v"(a.at[1][0]), "n"(OFF), "n"(OFF + 8 * RB) : "memory");
  } else if constexpr (DT == 2) {
    asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%8\n\t"
                 "ds_read_b64_tr_b16 %1, %5 offset:%9\n\t"
                 "ds_read_b64_tr_b16 %2, %6 offset:%8\n\t"
                 "ds_read_b64_tr_b16 %3, %7 offset:%9\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1])
                 : "v"(a.at[0][0]), "v"(a.at[1][0]),
                   "v"(a.at[0][1]), "v"(a.at[1][1]), "n"(OFF), "n"(OFF + 8 * RB) : "memory");
  } else if constexpr (DT == 3) {
    asm volatile("ds_read_b64_tr_b16 %0, %6 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %1, %7 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %2, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %5, %11 offset:%13\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2])
                 : "v"(a.at[0][0]), "v"(a.at[1][0]),
                   "v"(a.at[0][1]), "v"(a.at[1][1]),
                   "v"(a.at[0][2]), "v"(a.at[1][2]), "n"(OFF), "n"(OFF + 8 * RB) : "memory");
  } else {
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%16\n\t"
                 "ds_read_b64_tr_b16 %1, %9 offset:%17\n\t"
                 "ds_read_b64_tr_b16 %2, %10 offset:%16\n\t"
                 "ds_read_b64_tr_b16 %3, %11 offset:%17\n\t"
                 "ds_read_b64_tr_b16 %4, %12 offset:%16\n\t"
                 "ds_read_b64_tr_b16 %5, %13 offset:%17\n\t"
                 "ds_read_b64_tr_b16 %6, %14 offset:%16\n\t"
                 "ds_read_b64_tr_b16 %7, %15 offset:%17\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
                 : "v"(a.at[0][0]), "v"(a.at[1][0]),
                   "v"(a.at[0][1]), "v"(a.at[1][1]),
                   "v"(a.at[0][2]), "v"(a.at[1][2]),
                   "v"(a.at[0][3]), "v"(a.at[1][3]), "n"(OFF), "n"(OFF + 8 * RB) : "memory");
  }
#pragma unroll
  for (int d = 0; d < DT; ++d) f[d] = u32x4{lo[d][0], lo[d][1], hi[d][0], hi[d][1]};
}

// What every kernel of the family gets.  Strides in elements: batch, token, head.
struct XaArgs {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  float *lse, *lse2, *delta, *part, *part_lse;
  const int* lengths;
  const unsigned char* mask;
  long long qs[3], ks[3], vs[3], os[3], gs[3], dqs[3], dks[3], dvs[3], ms;
  int B, Lq, Lk, Hkv, G, D, rows, nsplit, tiles, nw, ragged;
  float scale;
};

// The block's share of the grid: blockIdx.x runs over (tile, split) of a (batch, key head).  Workgroups go to the 8 XCDs in
// turn; when the heads divide into whole rounds of 8, all blocks of a head run on one XCD, so that its keys and values are
// fetched into one L2.  (Dealing a head's blocks out to all XCDs where lengths are ragged evens their work out, and
// measured the same.)
__device__ __forceinline__ void xa_block(int per_head, int heads, int& inner, int& head) {
  const int id = blockIdx.x;
  if ((heads & 7) == 0) {
    const int xcd = id & 7, slot = id >> 3;
    head = (slot / per_head) * 8 + xcd;
    inner = slot % per_head;
  } else {
    head = id / per_head;
    inner = id % per_head;
  }
}
__device__ __forceinline__ int xa_keys(const XaArgs& A, int b) {
  int n = A.Lk;
  if (A.lengths) {
    const int m = A.lengths[b];
    n = m < 0 ? 0 : m < n ? m : n;
  }
  return n;
}
// bit i: key base + i counts (base + 64 keys, of which `n` exist, `byte` being this lane's mask byte)
__device__ __forceinline__ u64 xa_word(int n, bool masked, int byte) {
  u64 w = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
  if (masked) w &= __ballot(byte != 0);
  return w;
}

// host side, shared by the two files
int xa_check(const ried_xattn_t* d, const char* name, bool bwd);
XaArgs xa_args(const ried_xattn_t& d);
