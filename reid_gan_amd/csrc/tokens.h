// Element types shared by the token kernels (layer norm, rotary positions, cross attention, AdamW): fp32, bf16 and fp16 in
// memory, fp32 in registers.  A row may start anywhere its elements may: gfx950 reads 16 bytes from any element-aligned
// address, so odd widths need no path of their own, only a tail.
#pragma once
#include "common.h"

#define RIED_T_F32 0
#define RIED_T_BF16 1
#define RIED_T_F16 2

template <typename T> struct TokType;
template <> struct TokType<float> {
  static constexpr int V = 4;                                    // elements of 16 bytes
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct TokType<bf16_t> {
  static constexpr int V = 8;
  static __device__ __forceinline__ float up(bf16_t v) { return bf2f(v); }
  static __device__ __forceinline__ bf16_t down(float v) { return f2bf(v); }
};
template <> struct TokType<_Float16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 down(float v) { return (_Float16)v; }
};

// N consecutive elements at element alignment
template <typename T, int N> struct TokVec {
  T e[N];
} __attribute__((packed, aligned(sizeof(T))));

// Loads come in two steps - the elements as they lie, and their values - so that a kernel can have all its loads in
// flight before the first is used (a conversion inside the branch of a partial load would wait for it there).
template <typename T, int N>
__device__ __forceinline__ TokVec<T, N> tok_raw(const T* p) { return *reinterpret_cast<const TokVec<T, N>*>(p); }
// the first n of N (n <= 0: none); what is not there reads as zero
template <typename T, int N>
__device__ __forceinline__ TokVec<T, N> tok_raw_n(const T* p, int n) {
  TokVec<T, N> v;
  if (n >= N) {
    v = tok_raw<T, N>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v.e[i] = i < n ? p[i] : (T)0;
  }
  return v;
}
template <typename T, int N>
__device__ __forceinline__ void tok_up(const TokVec<T, N>& v, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = TokType<T>::up(v.e[i]);
}
template <typename T, int N>
__device__ __forceinline__ void tok_load_n(const T* p, int n, float (&f)[N]) { tok_up(tok_raw_n<T, N>(p, n), f); }
template <typename T, int N>
__device__ __forceinline__ void tok_store(T* p, const float (&f)[N]) {
  TokVec<T, N> v;
#pragma unroll
  for (int i = 0; i < N; ++i) v.e[i] = TokType<T>::down(f[i]);
  *reinterpret_cast<TokVec<T, N>*>(p) = v;
}
template <typename T, int N>
__device__ __forceinline__ void tok_store_n(T* p, int n, const float (&f)[N]) {
  if (n >= N) {
    tok_store<T, N>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = TokType<T>::down(f[i]);
  }
}

// sum over groups of L adjacent lanes (L a power of two up to 64), in every lane
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (L == 64) return wave_sum(v);
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

#define TOK_DISPATCH(type, T, ...)                              \
  switch (type) {                                               \
    case RIED_T_F32: { using T = float; __VA_ARGS__; break; }   \
    case RIED_T_BF16: { using T = bf16_t; __VA_ARGS__; break; } \
    default: { using T = _Float16; __VA_ARGS__; break; }        \
  }
static inline int tok_size(int type) { return type == RIED_T_F32 ? 4 : 2; }
static inline bool tok_type_ok(int type) { return type >= RIED_T_F32 && type <= RIED_T_F16; }
