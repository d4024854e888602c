// Tiles over 8-bit codes, gated, for each type of the results.
#include "projection_tile_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_tile_int8_gated(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s) {
  if (p.out_dtype == kF16) return launch_projection_tile<int8_t, _Float16, kProjGated, false, false>(p, bm, bn, deep, s);
  if (p.out_dtype == kBF16) return launch_projection_tile<int8_t, __bf16, kProjGated, false, false>(p, bm, bn, deep, s);
  return launch_projection_tile<int8_t, float, kProjGated, false, false>(p, bm, bn, deep, s);
}
}  // namespace cmpext3
