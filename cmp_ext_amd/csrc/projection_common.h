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

// A sum of codes times the scales of its row and column, the row's first, but last where it is large: a sum is below
// 2^31, so that no step leaves fp32's range where the result lies in it.  (The factors of 1 change nothing.)
struct RowScaled {
  float first, last;
  __device__ __forceinline__ explicit RowScaled(float scale) {
    const bool large = __builtin_fabsf(scale) > 0x1p60f;
    first = large ? 1.f : scale;
    last = large ? scale : 1.f;
  }
  __device__ __forceinline__ float operator()(float sum, float column) const { return sum * first * column * last; }
};

// f16 gradients: what undoes the unit of row m of entry bz's a (1 otherwise).  A power of two: the product with it is exact.
template <typename T, int MODE>
__device__ __forceinline__ float row_unit(const ProjParams& p, int bz, int64_t m) {
  if constexpr (std::is_same<T, _Float16>::value && MODE != kProjGated)
    return p.a_scale != nullptr ? p.a_scale[bz * (int64_t)p.M + m] : 1.f;
  return 1.f;
}

// 16 bytes at any address.
typedef u32x4 u32x4_any __attribute__((aligned(1)));

// v without its first `bytes` bytes (0 to 16), zeros behind.  In steps of 32 bits: with 64-bit shifts by a variable amount
// some waves' data were shifted by other amounts here, in 15 of 900 calls, right after memory was mapped; with these in none of
// 2700.  The amount lay in the last register a wave has (v15 of 16), which may be the cause; that was not shown.
__device__ __forceinline__ u32x4 drop_bytes(u32x4 v, int bytes) {
  const int words = bytes >> 2;
  if (words & 1) v = u32x4{v.y, v.z, v.w, 0};
  if (words & 2) v = u32x4{v.z, v.w, 0, 0};
  if (words & 4) v = u32x4{0, 0, 0, 0};
  const uint32_t by = (uint32_t)bytes & 3;
  return u32x4{__builtin_amdgcn_alignbyte(v.y, v.x, by), __builtin_amdgcn_alignbyte(v.z, v.y, by), __builtin_amdgcn_alignbyte(v.w, v.z, by),
               __builtin_amdgcn_alignbyte(0u, v.w, by)};
}

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

// Workgroup w runs on XCD w % 8: gives each XCD a contiguous range of the `total` strips of a matrix's rows,
// so that neighbouring rows are read from one XCD at a time (x[16, 8192] by 8192 rows of codes, 32 a strip: 19.2
// -> 12.4 us; x[1, 4096] by 4096 rows, 16 a strip: 6.1 -> 4.6).
__device__ __forceinline__ int strip_of(int w, int total) {
  const int xcd = w & 7, base = total >> 3, rem = total & 7;
  return xcd * base + (xcd < rem ? xcd : rem) + (w >> 3);
}

// LDS-DMA of dma_load16_m0 with the non-temporal policy, for what is read once.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <uint32_t DST>
__device__ __forceinline__ void dma_load16_m0_once(i32x4 rsrc, uint32_t voff, uint32_t soff, uint32_t lds_base,
                                                   std::integral_constant<uint32_t, DST> = {}) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen nt lds"
               :
               : "v"(voff), "s"(rsrc), "s"(lds_base + DST), "s"(soff)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// The end of the kernels for few rows: adds the sums of WAVES waves, [wave][16 MB rows of x][PITCH] of which the
// first 16 NB are a strip's rows (gated: 16 of w_gate, 16 of w_up, ..), and finishes and stores the results.
// a_scale: of x's rows, in memory or LDS.
template <typename T, int MODE, int MB, int NB, int WAVES, int PITCH>
__device__ __forceinline__ void finish_rows(const ProjParams& p, const void* red, int n0, const float* a_scale) {
  using E = typename std::conditional<sizeof(T) == 1, int, float>::type;
  constexpr bool GATED = MODE == kProjGated;
  constexpr int COLS = GATED ? 8 * NB : 16 * NB;
  const E* sums = (const E*)red;
  for (int o = threadIdx.x; o < 16 * MB * COLS; o += 64 * WAVES) {
    const int64_t m = o / COLS, n = n0 + o % COLS;
    if (m >= p.M || n >= p.N) continue;
    float v[2];
#pragma unroll
    for (int q = 0; q < (GATED ? 2 : 1); ++q) {
      const int c = GATED ? 32 * ((o % COLS) / 16) + 16 * q + o % 16 : o % COLS;
      E s = 0;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) s += sums[((i * MB * 16) + (int)m) * PITCH + c];
      v[q] = (float)s;
      if (sizeof(T) == 1) v[q] = RowScaled(a_scale[m])(v[q], p.b_scale[q][n]);
    }
    float y = v[0];
    if constexpr (GATED) {
      if (p.pre[0] != nullptr) {
        p.pre[0][m * p.ld_pre + n] = v[0];
        p.pre[1][m * p.ld_pre + n] = v[1];
      }
      with_act(p.act, [&](auto act) { y = act_value<decltype(act)::value>(v[0]) * v[1]; });
    } else if (p.bias != nullptr) {
      y += load_elem(p.bias, n, p.out_dtype);
    }
    store_elem(p.out[0], m * p.ldo[0] + n, p.out_dtype, y);
  }
}

}  // namespace cmpext3
