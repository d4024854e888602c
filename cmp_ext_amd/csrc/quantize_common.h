// Rows as 8-bit codes: a = max(max |x|, 2^-100), code = round(127 x / a), scale = a / 127.
#pragma once

#include "projection_common.h"

namespace cmpext3 {

// Eight elements as they are held between the passes.
template <typename T>
struct Piece {
  typedef u32x4 Any __attribute__((aligned(2)));
  u32x4 v;
  __device__ __forceinline__ void load(const T* x, int left) {
    if (left >= 8) {
      v = *(const Any*)x;
    } else {
      v = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) v[i >> 1] |= (uint32_t)((const uint16_t*)x)[i] << (16 * (i & 1));
    }
  }
  __device__ __forceinline__ float at(int i) const { return from_bits<T>((uint16_t)(v[i >> 1] >> (16 * (i & 1)))); }
};
template <>
struct Piece<float> {
  typedef f32x4 Any __attribute__((aligned(4)));
  f32x4 v[2];
  __device__ __forceinline__ void load(const float* x, int left) {
    if (left >= 8) {
      v[0] = *(const Any*)x;
      v[1] = *(const Any*)(x + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = i < left ? x[i] : 0.f;
    }
  }
  __device__ __forceinline__ float at(int i) const { return v[i >> 2][i & 3]; }
};

// The bits of the largest |x|: absolute values are ordered as their bits, infinity and NaN above all numbers.
template <typename T>
__device__ __forceinline__ uint32_t most_of(const Piece<T>& p, uint32_t a) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(p.at(i)) & 0x7fffffffu;
    a = a > b ? a : b;
  }
  return a;
}

// What the largest |x| of a row (its bits) makes of it.
struct RowScale {
  float up, a, inverse;  // 127, the largest value and its inverse, all times a unit
  float scale;
  uint32_t mask;  // of codes: none where the row is not finite
  __device__ __forceinline__ explicit RowScale(uint32_t most) {
    const bool finite = most < 0x7f800000u;
    const float amax = fmaxf(__uint_as_float(most), 0x1p-100f);
    // 127 x must not overflow: rows of large values are taken 2^-16 as large
    const float unit = amax > 0x1p100f ? 0x1p-16f : 1.f;
    up = 127.f * unit;
    a = amax * unit;
    inverse = 1.f / a;
    scale = finite ? amax / 127.f : __uint_as_float(0x7fc00000u);
    mask = finite ? ~0u : 0u;
  }
};

// Codes of four elements: round(127 x / a), a quotient by the inverse of a, corrected by what is left of 127 x
// (exactly, so that a quotient halfway between two codes is seen as that).  Adding 1.5 * 2^23 rounds to whole
// numbers, ties to even, and leaves them in the low bits.
template <typename T>
__device__ __forceinline__ uint32_t four_codes(const Piece<T>& p, int first, const RowScale& r) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = r.up * p.at(first + i), y = t * r.inverse;
    c[i] = __float_as_uint(fmaf(fmaf(-y, r.a, t), r.inverse, y) + 12582912.f);
  }
  const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
  return (lo | hi) & r.mask;
}

template <typename T>
__device__ __forceinline__ u32x2 eight_codes(const Piece<T>& p, const RowScale& r) {
  return u32x2{four_codes(p, 0, r), four_codes(p, 4, r)};
}

}  // namespace cmpext3
