// Rows as 8-bit codes with a scale for each: a = max(max |x|, 2^-100), code = round(127 x / a),
// scale = a / 127.  A workgroup takes a row: once for its largest value, once more for the codes.
#include "projection_common.h"

namespace cmpext3 {
namespace {

template <typename T>
__device__ __forceinline__ float as_float(const T* x, int64_t i) {
  return (float)x[i];
}

// round(127 x / a) for |x| <= a, inverse = 1 / a: a quotient by the inverse, corrected by what is left of
// 127 x (exactly, so that a quotient halfway between two codes is seen as that).
__device__ __forceinline__ int8_t code_of(float x, float a, float inverse) {
  const float t = 127.f * x;
  const float y = t * inverse;
  return (int8_t)(int)rintf(fmaf(fmaf(-y, a, t), inverse, y));
}

template <typename T>
__global__ void __launch_bounds__(256) quantize_int8_kernel(const QuantParams p) {
  __shared__ uint32_t most[4];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.x + row * p.ldx;
  // absolute values are ordered as their bits, with infinity and NaN above all numbers
  uint32_t a = 0;
  for (int i = threadIdx.x; i < p.cols; i += 256) {
    const uint32_t b = __float_as_uint(as_float(x, i)) & 0x7fffffffu;
    a = a > b ? a : b;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const uint32_t b = __shfl_xor(a, d);
    a = a > b ? a : b;
  }
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = a;
  __syncthreads();
  a = most[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) a = a > most[i] ? a : most[i];
  const bool finite = a < 0x7f800000u;
  const float amax = fmaxf(__uint_as_float(a), 0x1p-100f);
  // 127 x must not overflow: rows of large values are taken 2^-16 as large
  const float unit = amax > 0x1p100f ? 0x1p-16f : 1.f;
  const float most_x = amax * unit, inverse = 1.f / most_x;
  if (threadIdx.x == 0) p.scale[row] = finite ? amax / 127.f : __uint_as_float(0x7fc00000u);
  int8_t* codes = p.codes + row * p.ldc;
  for (int i = threadIdx.x; i < p.cols; i += 256) codes[i] = finite ? code_of(as_float(x, i) * unit, most_x, inverse) : (int8_t)0;
}

}  // namespace

hipError_t launch_quantize_int8(int dtype, const QuantParams& p, hipStream_t s) {
  const dim3 grid((unsigned)p.rows), block(256);
  if (dtype == kF16) return launch_kernel(quantize_int8_kernel<_Float16>, grid, block, 0, s, p);
  if (dtype == kBF16) return launch_kernel(quantize_int8_kernel<__bf16>, grid, block, 0, s, p);
  return launch_kernel(quantize_int8_kernel<float>, grid, block, 0, s, p);
}

}  // namespace cmpext3
