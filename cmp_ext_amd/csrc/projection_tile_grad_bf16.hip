// Tiles of a gated block's gradients, bf16: dx = dgate w_gate + dup w_up, and dw = d^T x.
#include "projection_tile_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_tile_sum_bf16(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s) {
  return launch_projection_tile<__bf16, __bf16, kProjSum, false, true>(p, bm, bn, deep, s);
}
hipError_t launch_projection_tile_wgrad_bf16(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s) {
  return launch_projection_tile<__bf16, __bf16, kProjPlain, true, true>(p, bm, bn, deep, s);
}
}  // namespace cmpext3
