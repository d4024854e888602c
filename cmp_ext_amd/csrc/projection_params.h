// Kernel arguments and launchers of the feed-forward operators, shared by the host planner
// and the device code.  Row pitches are in elements.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

namespace cmpext3 {

// Element types as in the C ABI (dtype codes of GemmParams, and 8-bit codes).
constexpr int kI8 = 4;

// What a kernel computes from its one or two products.
enum ProjMode : int {
  kProjPlain = 0,  // sum_k a b, scaled (8-bit codes), plus the bias
  kProjGated = 1,  // act(sum_k a b0) * (sum_k a b1)
  kProjSum = 2,    // sum_k a0 b0 + sum_k a1 b1
};

struct ProjParams {
  const void* a[2];  // kProjSum: both terms'; otherwise of each entry of the batch
  const void* b[2];  // kProjPlain: b[0]
  int64_t lda, ldb[2];
  const float* a_scale;     // 8-bit codes: of a row of a; f16 gradients: what undoes the units of a's rows, [batch][M], or nullptr
  const float* b_scale[2];  // 8-bit codes: of a row of b
  const void* bias;         // kProjPlain: [N] of the output's type, or nullptr
  void* out[2];  // of each entry of the batch
  int64_t ldo[2];
  int out_dtype;  // kF16, kBF16, kF32
  float* pre[2];  // kProjGated: both products, or nullptr
  int64_t ld_pre;
  int pre_vec;    // their rows are aligned to 16 bytes
  int act;
  int M, N, K;
  int batch;  // products with the same b (weight gradients: 2), else 1
  // tiles: their grid, rows of tiles of an ordering group, and splits of the steps of K (ksplit steps
  // each), whose sums go to partials [split][batch][product][M][ld_part]
  int tiles_m, tiles_n, group_m, splits, ksplit;
  void* partials;
  int64_t ld_part;
};

// Any pitch and alignment; a is [M, K] or, a_km, [K, M]; b is [N, K] or, b_kn, [K, N].
hipError_t launch_projection_any(int dtype, ProjMode mode, bool a_km, bool b_kn, const ProjParams& p, hipStream_t s);

// Up to kFewRows rows of a, b as [N, K], rows of whole 16 bytes.
constexpr int kFewRows = 64;
hipError_t launch_projection_rows(int dtype, ProjMode mode, const ProjParams& p, hipStream_t s);
// The same for few elements of x in 16 bits, which every workgroup makes codes of (lda: of x; a_scale: none).
constexpr int kRowsCodesRows = 16, kRowsCodesMost = 4096, kRowsCodesUnit = 512;  // rows, elements, of a row a multiple of
hipError_t launch_projection_rows_codes(int x_dtype, ProjMode mode, const ProjParams& p, hipStream_t s);

// Tiles of bm x bn = 256 x 256, 256 x 128 or 128 x 128; `deep` (128 x 128): alone on a CU, with a ring of four steps.  Operands have rows of
// whole 16 bytes.  (One translation unit for each element type and mode.)
using ProjTileLaunch = hipError_t(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s);
ProjTileLaunch launch_projection_tile_gated_f16, launch_projection_tile_gated_bf16;
ProjTileLaunch launch_projection_tile_sum_f16, launch_projection_tile_sum_bf16;
ProjTileLaunch launch_projection_tile_wgrad_f16, launch_projection_tile_wgrad_bf16;
ProjTileLaunch launch_projection_tile_int8_plain, launch_projection_tile_int8_gated;
// Tiles of 64 x 64, operands of any alignment whose rows have at least 16 bytes (sum and plain: see the modes' layouts
// above; gradients have a across k or b as [K, N] as the large tiles do).
// groups: 1 or 2 of four waves share a tile's steps.
using ProjSmallLaunch = hipError_t(ProjMode mode, const ProjParams& p, int groups, hipStream_t s);
ProjSmallLaunch launch_projection_small_f16, launch_projection_small_bf16, launch_projection_small_int8;
// Adds the splits' sums in their order and finishes the results as an unsplit kernel does.
hipError_t launch_projection_join(int dtype, ProjMode mode, const ProjParams& p, hipStream_t s);

// Rows copied to rows of whole 16 bytes, zeros behind row_bytes (16 at least); dst aligned to 16 bytes.
struct PadParams {
  struct Matrix {
    const void* src;
    void* dst;
    int64_t src_row, dst_row;  // bytes
    int rows, row_bytes;
  } m[3];
};
hipError_t launch_projection_pad(const PadParams& p, int count, hipStream_t s);

struct QuantParams {
  const void* x;
  int64_t ldx;
  int8_t* codes;
  int64_t ldc;
  float* scale;
  int64_t rows;
  int cols;
  int written;  // codes of a row: cols, or more, those past cols zeros
};
hipError_t launch_quantize_int8(int dtype, const QuantParams& p, hipStream_t s);

// Units of f16 gradients, powers of two: of a row of dgate and dup (for dx), of a column of either (for its weight).
struct GradUnits {
  float *row, *row_inverse;  // [M]
  float *col, *col_inverse;  // [2][ld_d], [2][N]
  // the largest finite values' bits: of rows within blocks of columns, of columns within blocks of rows
  uint32_t *row_most, *col_most;              // [col_blocks][M], [row_blocks][2][ld_d]
  int col_blocks, row_blocks, rows_of_block;  // see grad_blocks
};
constexpr int kGradBlockCols = 512;
// Blocks of rows: 128, or more where the columns are few, for 1024 workgroups; of 8 rows at least.
inline void grad_blocks(int64_t M, int64_t N, GradUnits* u) {
  u->col_blocks = (int)((N + kGradBlockCols - 1) / kGradBlockCols);
  const int64_t most = u->col_blocks < 8 ? 1024 / u->col_blocks : 128;
  u->rows_of_block = (int)(8 * ((M + 8 * most - 1) / (8 * most)));
  u->row_blocks = (int)((M + u->rows_of_block - 1) / u->rows_of_block);
}

// dgate = grad * up * act'(gate), dup = grad * act(gate): [M, N] each, rows of ld_d elements of
// which those past N are set to zero.
struct GatedGradParams {
  const void* grad;
  const float* gate;
  const float* up;
  void* d[2];      // dgate, dup: bf16 for all products; f16 for dx, rows times their units; or nullptr
  void* d_col[2];  // f16: for the weights, columns times their units; each or nullptr
  GradUnits units;
  int64_t ld_grad, ld_pre, ld_d;
  int act, M, N;
};
hipError_t launch_gated_grad(int dtype, const GatedGradParams& p, hipStream_t s);

}  // namespace cmpext3
