// Projections of few rows of x (generation: up to 64 tokens) by weights whose rows are whole 16 bytes: bound by
// reading the weights.
//
// A workgroup of four waves takes a strip of SW rows of the weights (gated: groups of 16 rows of w_gate and the
// same 16 of w_up) over all of K.  The strip and x's rows go global -> LDS by LDS-DMA through a ring of stages
// of RB bytes of k, so that HBM is read in runs of RB bytes and tens of KB are on their way in every CU
// without registers; LDS rows are XORed by row % 16, so that the fragment reads hit every bank once.  The
// waves split a stage's k and their sums are added in LDS at the end, where the activation, the
// scales and the bias follow.
//
// Where x is few elements of 16 bits and the weights are codes, every workgroup makes x's codes itself while its
// first stages are on their way, instead of a launch before: x[1, 4096] by 4096 rows of codes 8.8 -> 7.0 us, x[1, 2048], two
// of 2048 rows, 10.3 -> 7.0; but x[4, 4096] 11.4 for 9.1, so up to 4096 elements.
#pragma once

#include "quantize_common.h"

namespace cmpext3 {

// HELD: bytes of x's codes that are held for all of K; x is not part of the stages then.
template <int MB, int SW, int RB_, int NSMAX, int HELD>
struct ProjRowsShape {
  static constexpr int RB = RB_;
  static constexpr int W_BYTES = SW * RB, X_BYTES = HELD > 0 ? 0 : MB * 16 * RB;
  static constexpr int STAGE = W_BYTES + X_BYTES;
  static constexpr int FIT = (160 * 1024 - HELD) / STAGE;
  static constexpr int NS = FIT > NSMAX ? NSMAX : FIT;
  static constexpr int W_DMA = W_BYTES / 4096, X_DMA = X_BYTES / 4096;  // 1 KB loads of a wave and stage
  static constexpr int DMA = W_DMA + X_DMA;
  static constexpr int KB = RB / 64 / 4;  // products of a wave in k and stage
  static constexpr int PITCH = SW + 4;    // of the sums, four rows of a lane at a time
  static_assert(KB >= 1 && 1024 % RB == 0, "whole loads per row, products for every wave");
  static_assert(NS >= 3 && (NS - 2) * DMA <= 63, "ring depth / vmcnt range");
  static_assert(4 * MB * 16 * PITCH * 4 <= NS * STAGE, "the sums fit the ring");
};

// ONCE: the weights are read with the non-temporal policy.  X: the type of x, of which codes are made where it is not T.
template <typename T, int MODE, int MB, int SW, int RB, int NSMAX, bool ONCE, typename X = T>
__global__ void __launch_bounds__(256) projection_rows_kernel(const ProjParams p) {
  constexpr bool MAKE = !std::is_same<T, X>::value;
  using S = ProjRowsShape<MB, SW, RB, NSMAX, MAKE ? kRowsCodesMost : 0>;
  using Acc = typename Prod<T>::Acc;
  constexpr bool GATED = MODE == kProjGated;
  constexpr int NS = S::NS, NB = SW / 16, COLS = GATED ? SW / 2 : SW;
  static_assert(!GATED || NB % 2 == 0, "blocks of both weights");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[NS * S::STAGE];
  __shared__ __attribute__((aligned(1024))) unsigned char held[MAKE ? kRowsCodesMost : 16];
  __shared__ uint32_t most[16];
  __shared__ float scales[16];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = strip_of(blockIdx.x, gridDim.x) * COLS;
  const int bytes = p.K * (int)sizeof(T);

  // ---- DMA sources: load i of a wave is piece 4i + wave; 16-byte chunk c of row r lies at chunk c ^ (r % 16) ----
  auto geom = [&](int piece, int& row, int& at) {
    const int pos = piece * 1024 + 16 * lane;
    row = pos / RB;
    at = ((pos % RB) >> 4 ^ (row & 15)) * 16;
  };
  constexpr int XD = MAKE ? 1 : S::X_DMA;
  uint32_t w_off[S::W_DMA], x_off[XD];
  int w_at[S::W_DMA], x_at[XD];
#pragma unroll
  for (int i = 0; i < S::W_DMA; ++i) {
    int row;
    geom(4 * i + wave, row, w_at[i]);
    const int col = GATED ? (row >> 5) * 16 + (row & 15) : row;
    const int64_t ld = p.ldb[GATED ? (i * (4096 / RB) >> 4) & 1 : 0];
    w_off[i] = n0 + col < p.N ? (uint32_t)(col * ld * (int)sizeof(T) + w_at[i]) : kBufOOB;
  }
#pragma unroll
  for (int i = 0; i < (MAKE ? 0 : S::X_DMA); ++i) {
    int row;
    geom(4 * i + wave, row, x_at[i]);
    x_off[i] = row < p.M ? (uint32_t)(row * p.lda * (int)sizeof(T) + x_at[i]) : kBufOOB;
  }
  const i32x4 rx = make_rsrc_sgpr(MAKE ? nullptr : p.a[0]);
  i32x4 rw[2];
  rw[0] = make_rsrc_sgpr((const T*)p.b[0] + n0 * p.ldb[0]);
  rw[1] = GATED ? make_rsrc_sgpr((const T*)p.b[1] + n0 * p.ldb[1]) : rw[0];
#pragma unroll
  for (int i = 0; i < 2; ++i)  // in scalar registers, where the compiler would otherwise not always keep them
    rw[i][0] = __builtin_amdgcn_readfirstlane(rw[i][0]), rw[i][1] = __builtin_amdgcn_readfirstlane(rw[i][1]);
  auto load_stage = [&](int st) {
    const int k0 = st * RB, left = bytes - k0;  // pieces past the end load zeros and read no memory
    const uint32_t dst = lds_addr(smem) + (uint32_t)((st % NS) * S::STAGE + wave * 1024);
    static_for<S::W_DMA>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      constexpr int which = GATED ? (i * (4096 / RB) >> 4) & 1 : 0;
      const uint32_t voff = w_at[i] < left ? w_off[i] : kBufOOB;
      if constexpr (ONCE)
        dma_load16_m0_once(rw[which], voff, (uint32_t)k0, dst, std::integral_constant<uint32_t, i * 4096>{});
      else
        dma_load16_m0(rw[which], voff, (uint32_t)k0, dst, std::integral_constant<uint32_t, i * 4096>{});
    });
    static_for<MAKE ? 0 : S::X_DMA>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      const uint32_t voff = x_at[i] < left ? x_off[i] : kBufOOB;
      dma_load16_m0(rx, voff, (uint32_t)k0, dst, std::integral_constant<uint32_t, S::W_BYTES + i * 4096>{});
    });
  };

  const int c = lane & 15, g = lane >> 4;
  Acc acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB * MB; ++i) acc[i / MB][i % MB] = Prod<T>::zero();
  auto multiply_stage = [&](int st) {
    const unsigned char* w = smem + (st % NS) * S::STAGE;
    const unsigned char* x = MAKE ? held + min(c, p.M - 1) * bytes + st * RB : w + S::W_BYTES;
#pragma unroll
    for (int b = 0; b < S::KB; ++b) {
      const int at = 16 * (((wave * S::KB + b) * 4 + g) ^ c);
      const int at_x = 16 * (((wave * S::KB + b) * 4 + g) ^ min(c, p.M - 1));  // rows past the last one: the last
      u32x4 fx[MB];
#pragma unroll
      for (int m = 0; m < MB; ++m) fx[m] = *(const u32x4*)(x + (MAKE ? at_x : (16 * m + c) * RB + at));
#pragma unroll
      for (int h = 0; h < NB; ++h) {
        const u32x4 fw = *(const u32x4*)(w + (16 * h + c) * RB + at);
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[h][m] = Prod<T>::mma(fw, fx[m], acc[h][m]);
      }
    }
  };
  const int stages = (bytes + RB - 1) / RB;
  // x's elements are on their way before the stages: loads are waited for in their order
  constexpr int PER = kRowsCodesMost / 2048;  // pieces of 8 of a thread
  Piece<typename std::conditional<MAKE, X, _Float16>::type> px[MAKE ? PER : 1];
  const int row_pieces = p.K / 8, pieces = p.M * row_pieces;  // K is a multiple of 512: a wave's pieces are of one row
  if constexpr (MAKE) {
    if (tid < 16) most[tid] = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int q = 256 * i + 64 * wave;
      if (q < pieces) {
        const int m = q / row_pieces;
        px[i].load((const X*)p.a[0] + m * p.lda + 8 * (int64_t)(q - m * row_pieces + lane), 8);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int t = 0; t < NS - 1; ++t) load_stage(t);
  if constexpr (MAKE) {
    // the compiler's wait for x knows nothing of the stages' loads behind it, and waits for them too
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");  // `most` is zero
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int q = 256 * i + 64 * wave;
      if (q >= pieces) continue;
      uint32_t a = most_of(px[i], 0u);
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        const uint32_t b = __shfl_xor(a, d);
        a = a > b ? a : b;
      }
      if (lane == 0) atomicMax(&most[q / row_pieces], a);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
    if (tid < p.M) scales[tid] = RowScale(most[tid]).scale;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int q = 256 * i + 64 * wave;
      if (q >= pieces) continue;
      const int m = q / row_pieces, at = 8 * (q - m * row_pieces + lane);
      const int chunk = (at >> 4) ^ (m & 15);  // as the stages' rows are
      *(u32x2*)(held + m * bytes + 16 * chunk + (at & 8)) = eight_codes(px[i], RowScale(most[m]));
    }
  }
  ring_fence<(NS - 2) * S::DMA>();
  for (int st = 0; st < stages; ++st) {
    load_stage(st + NS - 1);
    multiply_stage(st);
    ring_fence<(NS - 2) * S::DMA>();
  }
  ring_fence<0>();

  // ---- the waves' sums: acc[h][m] holds x's row 16m + c with rows 4g .. 4g+3 of block h ----
  Acc* red = (Acc*)smem;
#pragma unroll
  for (int h = 0; h < NB; ++h)
#pragma unroll
    for (int m = 0; m < MB; ++m) red[((wave * MB + m) * 16 + c) * (S::PITCH / 4) + 4 * h + g] = acc[h][m];
  __syncthreads();
  finish_rows<T, MODE, MB, NB, 4, S::PITCH>(p, smem, n0, MAKE ? scales : p.a_scale);
}

// Strips, stages and rings, so that two workgroups (96 KB: one) share a CU where there are that many strips.
// MI355X, weights from HBM (us; ring of three, or as many as named):
//   x[16, 4096], two weights of 14336 rows, bf16: strips of 32 rows in runs of 512 bytes 40.1 (ring of four, one
//     workgroup per CU: 44.2; strips of 64 in runs of 256: 39.4); codes, x[4, 4096]: 22.9 and 24.6
//   x[16, 8192] by 8192 rows of codes: strips of 32 12.4, of 16 13.7, of 64 (half the CUs) 16.5
//   x[1, 4096] by 4096 rows of codes: strips of 16, ring of four 4.6, of 32 (half the CUs) 5.4
//   x[32, 4096], two of 14336, bf16: strips of 64 in runs of 256 41.9, of 32 in runs of 512 49.5
//   x[64, 4096], two of 14336, bf16: strips of 64 in runs of 256 52.3, of 32 in runs of 256 59.4, of 512 64.3
//   x[64, 8192] by 8192 rows of codes: strips of 32 in runs of 512 18.5, of 16 in runs of 256 24.5
// so: strips of 64 rows for more than 16 rows of x where they fill the CUs, else of 32, else (one weight) of 16.
template <typename T, int MODE, bool ONCE>
hipError_t launch_projection_rows_k(const ProjParams& p, hipStream_t s) {
  const int strips32 = (p.N + (MODE == kProjGated ? 15 : 31)) / (MODE == kProjGated ? 16 : 32);
  const dim3 block(256);
  auto go = [&](auto kernel, int cols) { return launch_kernel(kernel, dim3((unsigned)((p.N + cols - 1) / cols)), block, 0, s, p); };
  constexpr int HALF = MODE == kProjGated ? 2 : 1;
  if constexpr (MODE == kProjPlain) {
    if (strips32 < 256) {
      if (p.M <= 16) return go(projection_rows_kernel<T, MODE, 1, 16, 512, 4, ONCE>, 16);
      if (p.M <= 32) return go(projection_rows_kernel<T, MODE, 2, 16, 512, 3, ONCE>, 16);
      if (strips32 < 128) return go(projection_rows_kernel<T, MODE, 4, 16, 256, 4, ONCE>, 16);
    }
  }
  if (p.M <= 16) return go(projection_rows_kernel<T, MODE, 1, 32, 512, 3, ONCE>, 32 / HALF);
  if (strips32 < 512) {
    if (p.M <= 32) return go(projection_rows_kernel<T, MODE, 2, 32, 512, 3, ONCE>, 32 / HALF);
    return go(projection_rows_kernel<T, MODE, 4, 32, 512, 3, ONCE>, 32 / HALF);
  }
  if (p.M <= 32) return go(projection_rows_kernel<T, MODE, 2, 64, 256, 3, ONCE>, 64 / HALF);
  return go(projection_rows_kernel<T, MODE, 4, 64, 256, 3, ONCE>, 64 / HALF);
}

// The same strips with codes made of x.
template <typename X, int MODE, bool ONCE>
hipError_t launch_projection_rows_codes_k(const ProjParams& p, hipStream_t s) {
  constexpr int HALF = MODE == kProjGated ? 2 : 1;
  if constexpr (MODE == kProjPlain) {
    if ((p.N + 31) / 32 < 256)
      return launch_kernel((projection_rows_kernel<int8_t, MODE, 1, 16, 512, 4, ONCE, X>), dim3((unsigned)((p.N + 15) / 16)), dim3(256), 0, s, p);
  }
  const int cols = 32 / HALF;
  return launch_kernel((projection_rows_kernel<int8_t, MODE, 1, 32, 512, 3, ONCE, X>), dim3((unsigned)((p.N + cols - 1) / cols)), dim3(256), 0, s, p);
}

// Weights of 64 MB and more are read past the reusable lines: smaller ones may still be in the Infinity Cache at the
// next call (those above: 12.4 for 13.7, 40.1 for 43.9, 22.9 for 25.4; but x[1, 4096] by 4096 rows 5.0 for 4.6).
inline bool read_once(const ProjParams& p, int mode, int esz) { return (int64_t)p.N * p.K * esz * (mode == kProjGated ? 2 : 1) >= 64ll << 20; }
template <typename T, int MODE>
hipError_t launch_projection_rows(const ProjParams& p, hipStream_t s) {
  return read_once(p, MODE, sizeof(T)) ? launch_projection_rows_k<T, MODE, true>(p, s) : launch_projection_rows_k<T, MODE, false>(p, s);
}
template <typename X, int MODE>
hipError_t launch_projection_rows_codes(const ProjParams& p, hipStream_t s) {
  return read_once(p, MODE, 1) ? launch_projection_rows_codes_k<X, MODE, true>(p, s) : launch_projection_rows_codes_k<X, MODE, false>(p, s);
}

}  // namespace cmpext3
