// Gated tiles, bf16.
#include "projection_tile_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_tile_gated_bf16(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s) {
  return launch_projection_tile<__bf16, __bf16, kProjGated, false, false>(p, bm, bn, deep, s);
}
}  // namespace cmpext3
