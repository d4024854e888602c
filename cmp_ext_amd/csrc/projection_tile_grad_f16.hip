// Tiles of a gated block's gradients, f16: dx = dgate w_gate + dup w_up, and dw = d^T x.
#include "projection_tile_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_tile_sum_f16(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s) {
  return launch_projection_tile<_Float16, _Float16, kProjSum, false, true>(p, bm, bn, deep, s);
}
hipError_t launch_projection_tile_wgrad_f16(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s) {
  return launch_projection_tile<_Float16, _Float16, kProjPlain, true, true>(p, bm, bn, deep, s);
}
}  // namespace cmpext3
