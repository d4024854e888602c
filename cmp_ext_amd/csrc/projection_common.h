// What the kernels of the feed-forward operators share: products on 16-byte fragments of any
// element type, and stores of any output type.
#pragma once

#include "activation.h"
#include "device_common.h"
#include "projection_params.h"

namespace cmpext3 {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

// A product of 16 x 16 results over 64 bytes of k: lane l supplies 16 bytes of row l % 16 at byte
// 16 (l / 16) of both operands, so that LDS rows and fragments look alike for 16-bit elements
// (32 k) and for codes (64 k).  The first operand's rows are output columns, as in Mfma<T>.
template <typename T>
struct Prod {
  using Acc = f32x4;
  static __device__ __forceinline__ Acc zero() { return Acc{0.f, 0.f, 0.f, 0.f}; }
  static __device__ __forceinline__ Acc mma(u32x4 b, u32x4 a, Acc c) { return Mfma<T>::mma(b, a, c); }
};
template <>
struct Prod<int8_t> {
  using Acc = i32x4_t;
  static __device__ __forceinline__ Acc zero() { return Acc{0, 0, 0, 0}; }
  static __device__ __forceinline__ Acc mma(u32x4 b, u32x4 a, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, b), __builtin_bit_cast(i32x4_t, a), c, 0, 0, 0);
  }
};

// One element of the given type (kF16, kBF16, kF32), rounded to nearest even.
__device__ __forceinline__ void store_elem(void* base, int64_t i, int dtype, float v) {
  if (dtype == kF32)
    ((float*)base)[i] = v;
  else
    ((uint16_t*)base)[i] = dtype == kF16 ? to_bits<_Float16>(v) : to_bits<__bf16>(v);
}
__device__ __forceinline__ float load_elem(const void* base, int64_t i, int dtype) {
  if (dtype == kF32) return ((const float*)base)[i];
  const uint16_t h = ((const uint16_t*)base)[i];
  return dtype == kF16 ? from_bits<_Float16>(h) : from_bits<__bf16>(h);
}

}  // namespace cmpext3
