// Small tiles over 8-bit codes.
#include "projection_small_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_small_int8(ProjMode mode, const ProjParams& p, int groups, hipStream_t s) {
  if (mode == kProjGated) return launch_projection_small<int8_t, kProjGated, false, false>(p, groups, s);
  return launch_projection_small<int8_t, kProjPlain, false, false>(p, groups, s);
}
}  // namespace cmpext3
