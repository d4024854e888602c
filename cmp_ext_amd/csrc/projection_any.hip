// Products of the feed-forward operators for any size, pitch and alignment, an element at a time: for what the others
// cannot take, rows of less than 16 bytes, no k at all, and grids beyond theirs.  (Codes, 4096 x 4096 x 14336: 2031 us.)
//
// One workgroup of four waves sums a 64 x 64 block of results in steps of 64 bytes of k (32
// 16-bit elements, 64 codes).  Operands go through registers into LDS rows of one row's (or
// column's) k, so that either may lie along k or across it; neighbouring lanes read neighbouring
// elements in both cases.
#include "projection_common.h"

namespace cmpext3 {
namespace {

constexpr int kAnyTile = 64;
constexpr int kAnyPitch = 80;  // bytes of an LDS row: 64 of k, and 16 that spread rows over the banks

// src is [rows, K] (or [K, rows] if KM): rows row0 .. + 63 at k0 .. + KS - 1, zeros outside.
template <typename E, bool KM>
__device__ __forceinline__ void any_load(unsigned char* lds, const E* src, int64_t ld, int rows, int row0, int K, int k0) {
  constexpr int KS = 64 / sizeof(E);
  constexpr int PER = kAnyTile * KS / 256;
  E v[PER];
  int at[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = threadIdx.x + 256 * i;
    const int r = KM ? e % kAnyTile : e / KS, k = KM ? e / kAnyTile : e % KS;
    at[i] = r * kAnyPitch + k * (int)sizeof(E);
    const int64_t row = (int64_t)row0 + r, kk = (int64_t)k0 + k;
    v[i] = row < rows && kk < K ? src[KM ? kk * ld + row : row * ld + kk] : (E)0;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) *(E*)(lds + at[i]) = v[i];
}

template <typename T, int MODE, bool A_KM, bool B_KN>
__global__ void __launch_bounds__(256) projection_any_kernel(const ProjParams p) {
  using E = typename std::conditional<sizeof(T) == 1, int8_t, uint16_t>::type;
  constexpr int KS = 64 / sizeof(T);
  constexpr int NP = MODE == kProjGated ? 2 : 1;  // products held at once
  __shared__ __attribute__((aligned(16))) unsigned char sa[kAnyTile * kAnyPitch], sb[NP][kAnyTile * kAnyPitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, G = lane >> 4;
  const int m0 = blockIdx.x * kAnyTile, n0 = blockIdx.y * kAnyTile;
  const int wm = 32 * (wave >> 1), wn = 32 * (wave & 1);
  typename Prod<T>::Acc acc[NP][2][2];
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[q][i >> 1][i & 1] = Prod<T>::zero();
#pragma unroll
  for (int part = 0; part < (MODE == kProjSum ? 2 : 1); ++part) {
    const E* a = (const E*)p.a[MODE == kProjSum ? part : blockIdx.z];
    for (int k0 = 0; k0 < p.K; k0 += KS) {
      __syncthreads();
      any_load<E, A_KM>(sa, a, p.lda, p.M, m0, p.K, k0);
#pragma unroll
      for (int q = 0; q < NP; ++q) any_load<E, B_KN>(sb[q], (const E*)p.b[part + q], p.ldb[part + q], p.N, n0, p.K, k0);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32x4 fa = *(const u32x4*)(sa + (wm + 16 * i + r16) * kAnyPitch + 16 * G);
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u32x4 fb = *(const u32x4*)(sb[q] + (wn + 16 * j + r16) * kAnyPitch + 16 * G);
            acc[q][i][j] = Prod<T>::mma(fb, fa, acc[q][i][j]);
          }
      }
    }
  }
  // acc[q][i][j][e]: row 16i + r16, column 16j + 4G + e of the wave's block
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + wm + 16 * i + r16;
    if (m >= p.M) continue;
    const float as = sizeof(T) == 1 ? p.a_scale[m] : row_unit<T, MODE>(p, blockIdx.z, m);
    const RowScaled scaled(as);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int j = x >> 2, e = x & 3;
      const int64_t n = n0 + wn + 16 * j + 4 * G + e;
      if (n >= p.N) continue;
      float v[NP];
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        v[q] = (float)acc[q][i][j][e];
        if (sizeof(T) == 1) v[q] = scaled(v[q], p.b_scale[q][n]);
        else v[q] *= as;
      }
      float y = v[0];
      if constexpr (MODE == kProjGated) {
        if (p.pre[0] != nullptr) {
          p.pre[0][m * p.ld_pre + n] = v[0];
          p.pre[1][m * p.ld_pre + n] = v[1];
        }
        with_act(p.act, [&](auto act) { y = act_value<decltype(act)::value>(v[0]) * v[1]; });
      } else if (p.bias != nullptr) {
        y += load_elem(p.bias, n, p.out_dtype);
      }
      store_elem(p.out[blockIdx.z], m * p.ldo[blockIdx.z] + n, p.out_dtype, y);
    }
  }
}

template <typename T>
hipError_t launch16(ProjMode mode, bool a_km, bool b_kn, const ProjParams& p, dim3 grid, hipStream_t s) {
  if (mode == kProjGated && !a_km && !b_kn)
    return launch_kernel((projection_any_kernel<T, kProjGated, false, false>), grid, dim3(256), 0, s, p);
  if (mode == kProjSum && !a_km && b_kn)
    return launch_kernel((projection_any_kernel<T, kProjSum, false, true>), grid, dim3(256), 0, s, p);
  if (mode == kProjPlain && a_km && b_kn)
    return launch_kernel((projection_any_kernel<T, kProjPlain, true, true>), grid, dim3(256), 0, s, p);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_projection_any(int dtype, ProjMode mode, bool a_km, bool b_kn, const ProjParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.M + kAnyTile - 1) / kAnyTile), (unsigned)((p.N + kAnyTile - 1) / kAnyTile), (unsigned)p.batch);
  if (dtype == kF16) return launch16<_Float16>(mode, a_km, b_kn, p, grid, s);
  if (dtype == kBF16) return launch16<__bf16>(mode, a_km, b_kn, p, grid, s);
  if (mode == kProjPlain) return launch_kernel((projection_any_kernel<int8_t, kProjPlain, false, false>), grid, dim3(256), 0, s, p);
  return launch_kernel((projection_any_kernel<int8_t, kProjGated, false, false>), grid, dim3(256), 0, s, p);
}

}  // namespace cmpext3
