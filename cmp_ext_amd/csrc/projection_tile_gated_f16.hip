// Gated tiles, f16.
#include "projection_tile_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_tile_gated_f16(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s) {
  return launch_projection_tile<_Float16, _Float16, kProjGated, false, false>(p, bm, bn, deep, s);
}
}  // namespace cmpext3
