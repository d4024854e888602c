// Projections of few rows of x (up to 64) by weights whose rows are not whole 16 bytes, which LDS-DMA cannot
// take.
//
// One workgroup takes NB blocks of 16 rows of the weights (gated: 16 of each) over all of K; its waves take
// steps of 128 bytes of k in turn, so that a row is read in runs of whole lines.  The instruction's own
// layout is what a lane loads: 16 bytes of row l % 16 at byte 16 (l / 16) of every 64, from memory straight
// into registers, weights and x alike, DEPTH steps ahead.  Rows may start at any element; what the last 16 bytes of
// a row hold past its end is shifted out.  Rows past the last one are read as the last one and not stored.
// Bound by the rate at which a CU takes in lines in pieces of 64 bytes, x's among them: x[16, 4096] with two weights
// of 14336 rows of bf16 48.5 us (through LDS 40.1), x[64, 4096] 94 (52).
#pragma once

#include "projection_common.h"

namespace cmpext3 {

typedef u32x4 u32x4_any __attribute__((aligned(1)));

// 16 bytes from any address.
__device__ __forceinline__ u32x4 load16_any(const char* p) { return *(const u32x4_any*)p; }

// The 16 bytes at `at` of a row of `bytes` >= 16, zeros past its end: loaded from where they end with the row, and
// shifted.
__device__ __forceinline__ u32x4 load16_end(const char* row, int64_t at, int64_t bytes) {
  const int64_t over = at + 16 - bytes;
  if (over >= 16) return u32x4{0, 0, 0, 0};
  if (over <= 0) return load16_any(row + at);
  const u32x4 v = load16_any(row + bytes - 16);
  unsigned __int128 x = __builtin_bit_cast(unsigned __int128, v);
  x >>= 8 * (int)over;
  return __builtin_bit_cast(u32x4, x);
}

// MB: 16-row blocks of x; NB: of the weights (gated: one of each); W: waves.
template <typename T, int MODE, int MB, int NB, int W, int DEPTH>
__global__ void __launch_bounds__(64 * W) projection_rows_any_kernel(const ProjParams p) {
  using Acc = typename Prod<T>::Acc;
  constexpr bool GATED = MODE == kProjGated;
  constexpr int COLS = GATED ? 16 * (NB / 2) : 16 * NB;  // results of a workgroup in a row
  constexpr int PITCH = 16 * NB + 4;                     // of the sums in LDS
  __shared__ __attribute__((aligned(16))) Acc red[W * MB * 16 * PITCH / 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, G = lane >> 4;
  const int n0 = strip_of(blockIdx.x, gridDim.x) * COLS;
  const int64_t bytes = (int64_t)p.K * (int)sizeof(T);
  const char* w[NB];
  const char* x[MB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int which = GATED ? b & 1 : 0;
    const int row = min(n0 + 16 * (GATED ? b >> 1 : b) + r16, p.N - 1);
    w[b] = (const char*)p.b[which] + row * p.ldb[which] * (int64_t)sizeof(T);
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) x[b] = (const char*)p.a[0] + min(16 * b + r16, p.M - 1) * p.lda * (int64_t)sizeof(T);

  Acc acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB * MB; ++i) acc[i / MB][i % MB] = Prod<T>::zero();
  const int steps = (int)(bytes / 128);  // whole ones; the wave whose turn comes then takes the rest
  u32x4 fw[DEPTH][NB][2], fx[DEPTH][MB][2];
  auto load = [&](int d, int step) {
    const int64_t at = (int64_t)step * 128 + 16 * G;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int b = 0; b < NB; ++b) fw[d][b][s] = load16_any(w[b] + at + 64 * s);
#pragma unroll
      for (int b = 0; b < MB; ++b) fx[d][b][s] = load16_any(x[b] + at + 64 * s);
    }
  };
  auto multiply = [&](int d) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[b][m] = Prod<T>::mma(fw[d][b][s], fx[d][m][s], acc[b][m]);
  };
  // DEPTH steps are on their way while one is multiplied.  The barriers keep that order: left to itself the
  // compiler moves loads behind the products of later steps.
  const int mine = steps > wave ? (steps - wave + W - 1) / W : 0;  // of this wave: steps wave, wave + W, ..
  if (mine > 0) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(d, wave + W * min(d, mine - 1));
    int i = 0;
    for (; i + 2 * DEPTH <= mine; i += DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        multiply(d);
        load(d, wave + W * (i + d + DEPTH));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (i + d < mine) multiply(d);
      if (i + d + DEPTH < mine) load(d, wave + W * (i + d + DEPTH));
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
      if (i + d + DEPTH < mine) multiply(d);
  }
  if (steps * (int64_t)128 < bytes && steps % W == wave) {
    const int64_t at = (int64_t)steps * 128 + 16 * G;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int b = 0; b < NB; ++b) fw[0][b][s] = load16_end(w[b], at + 64 * s, bytes);
#pragma unroll
      for (int b = 0; b < MB; ++b) fx[0][b][s] = load16_end(x[b], at + 64 * s, bytes);
    }
    multiply(0);
  }

  // ---- sums of the waves: acc[b][m] holds x's row 16m + r16 with rows 4G .. 4G+3 of block b ----
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int m = 0; m < MB; ++m) red[((wave * MB + m) * 16 + r16) * (PITCH / 4) + 4 * b + G] = acc[b][m];
  __syncthreads();
  finish_rows<T, MODE, MB, NB, W, PITCH>(p, red, n0);
}

// Eight waves, two steps ahead, 32 rows of the weights (16 of one that does not fill the CUs).
template <typename T, int MODE, int MB>
hipError_t launch_projection_rows_any_k(const ProjParams& p, hipStream_t s) {
  const dim3 block(512);
  if (MODE == kProjPlain && p.N > 32 * 256)
    return launch_kernel((projection_rows_any_kernel<T, MODE, MB, 2, 8, 2>), dim3((unsigned)((p.N + 31) / 32)), block, 0, s, p);
  return launch_kernel((projection_rows_any_kernel<T, MODE, MB, MODE == kProjGated ? 2 : 1, 8, 2>), dim3((unsigned)((p.N + 15) / 16)), block, 0, s, p);
}
template <typename T, int MODE>
hipError_t launch_projection_rows_any(const ProjParams& p, hipStream_t s) {
  if (p.M <= 16) return launch_projection_rows_any_k<T, MODE, 1>(p, s);
  if (p.M <= 32) return launch_projection_rows_any_k<T, MODE, 2>(p, s);
  return launch_projection_rows_any_k<T, MODE, 4>(p, s);
}

}  // namespace cmpext3
