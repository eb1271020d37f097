// Row-wise loads and stores of 16-byte pieces with a ragged end, shared by the layer-norm and gradient-norm kernels.
#pragma once
#include "common.h"

typedef _Float16 f16_t;

// values of one 16-byte piece
template <typename T> struct Piece { static constexpr int V = 16 / sizeof(T); };

// p[0 .. n - 1] as fp32, zeros behind; p is aligned to its type only (one dwordx4 in the target's unaligned mode)
template <typename T>
__device__ __forceinline__ void load_piece(const T *p, int n, float (&v)[Piece<T>::V]) {
  constexpr int V = Piece<T>::V;
  if (n >= V) {
    T e[V];
    __builtin_memcpy(e, p, 16);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = (float)e[k];
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = k < n ? (float)p[k] : 0.f;
  }
}
// the same piece as it lies in memory (for loads that are to be under way while something else is computed), and its values
template <typename T>
__device__ __forceinline__ u32x4 load_raw(const T *p, int n) {
  constexpr int V = Piece<T>::V;
  u32x4 r = {0u, 0u, 0u, 0u};
  if (n >= V) {
    __builtin_memcpy(&r, p, 16);
  } else if (n > 0) {
    T e[V];
#pragma unroll
    for (int k = 0; k < V; ++k) e[k] = k < n ? p[k] : (T)0.f;
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void raw_values(u32x4 r, float (&v)[Piece<T>::V]) {
  constexpr int V = Piece<T>::V;
  T e[V];
  __builtin_memcpy(e, &r, 16);
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = (float)e[k];
}
// V values of a vector of another type (layer-norm weights beside 16-bit rows)
template <typename S, int V>
__device__ __forceinline__ void load_values(const S *p, int n, float (&v)[V]) {
  if (n >= V) {
    S e[V];
    __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = (float)e[k];
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = k < n ? (float)p[k] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_piece(T *p, int n, const float (&v)[Piece<T>::V]) {
  constexpr int V = Piece<T>::V;
  if (n >= V) {
    T e[V];
#pragma unroll
    for (int k = 0; k < V; ++k) e[k] = (T)v[k];
    __builtin_memcpy(p, e, 16);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) p[k] = (T)v[k];
  }
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}
