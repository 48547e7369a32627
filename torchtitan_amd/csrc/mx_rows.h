// Rows of bf16 (as uint16_t) or float32 elements, read and written in pieces of V elements from any element on:
// the hardware takes 16-byte accesses at any element's address, so rows of odd lengths and views that start
// anywhere need no copies.  A piece that the row ends in is read and written element by element.
#pragma once

#include <type_traits>

#include "mx_common.h"

namespace mx {

typedef uint32_t u32x4_el2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_el4 __attribute__((ext_vector_type(4), aligned(4)));

// V elements of T as they lie in memory: 16 bytes or 32.
template <class T, int V>
struct Piece {
  static constexpr int kWords = V * (int)sizeof(T) / 4;
  uint32_t w[kWords];
};

template <bool NT, class T, int V>
__device__ __forceinline__ void load_words(const T* p, Piece<T, V>& q) {
  using W = std::conditional_t<sizeof(T) == 4, u32x4_el4, u32x4_el2>;
#pragma unroll
  for (int k = 0; k < Piece<T, V>::kWords / 4; ++k) {
    const W* s = reinterpret_cast<const W*>(p) + k;
    const W v = NT ? __builtin_nontemporal_load(s) : *s;
    q.w[4 * k] = v.x, q.w[4 * k + 1] = v.y, q.w[4 * k + 2] = v.z, q.w[4 * k + 3] = v.w;
  }
}
template <bool NT, class T, int V>
__device__ __forceinline__ void store_words(T* p, const Piece<T, V>& q) {
  using W = std::conditional_t<sizeof(T) == 4, u32x4_el4, u32x4_el2>;
#pragma unroll
  for (int k = 0; k < Piece<T, V>::kWords / 4; ++k) {
    W* d = reinterpret_cast<W*>(p) + k;
    const W v = {q.w[4 * k], q.w[4 * k + 1], q.w[4 * k + 2], q.w[4 * k + 3]};
    if (NT) __builtin_nontemporal_store(v, d); else *d = v;
  }
}

// The piece at p of which `left` elements belong to the row (fewer than one: none); the others read as 0.
template <bool NT, class T, int V>
__device__ __forceinline__ void load_piece(const T* p, int64_t left, Piece<T, V>& q) {
  if (left >= V) {
    load_words<NT>(p, q);
    return;
  }
#pragma unroll
  for (int k = 0; k < Piece<T, V>::kWords; ++k) q.w[k] = 0;
#pragma unroll
  for (int e = 0; e < V - 1; ++e)
    if (e < left) {
      if constexpr (sizeof(T) == 4) q.w[e] = __float_as_uint(p[e]);
      else q.w[e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
    }
}
template <bool NT, class T, int V>
__device__ __forceinline__ void store_piece(T* p, int64_t left, const Piece<T, V>& q) {
  if (left >= V) {
    store_words<NT>(p, q);
    return;
  }
#pragma unroll
  for (int e = 0; e < V - 1; ++e)
    if (e < left) {
      if constexpr (sizeof(T) == 4) p[e] = __uint_as_float(q.w[e]);
      else p[e] = (uint16_t)(q.w[e / 2] >> (16 * (e & 1)));
    }
}

template <class T, int V>
__device__ __forceinline__ void to_floats(const Piece<T, V>& q, float (&f)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (sizeof(T) == 4) f[e] = __uint_as_float(q.w[e]);
    else f[e] = e & 1 ? bf16_hi(q.w[e / 2]) : bf16_lo(q.w[e / 2]);
  }
}
// To bf16 to nearest even (v_cvt_pk_bf16_f32: NaN stays NaN): the one rounding of a result held in float32.
template <class T, int V>
__device__ __forceinline__ Piece<T, V> from_floats(const float (&f)[V]) {
  Piece<T, V> q;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) q.w[e] = __float_as_uint(f[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2)
      q.w[e / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f_t{f[e], f[e + 1]}, v2bf_t));
  }
  return q;
}

// Lane exchange inside 16 lanes (see dpp): lane i from lane 15 - i; of 8, from lane 7 - i.
constexpr int kRowMirror = 0x140, kRowHalfMirror = 0x141;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

}  // namespace mx
