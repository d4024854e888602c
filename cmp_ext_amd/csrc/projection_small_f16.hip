// Small tiles of a gated block and its gradients, f16.
#include "projection_small_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_small_f16(ProjMode mode, const ProjParams& p, int groups, hipStream_t s) {
  if (mode == kProjGated) return launch_projection_small<_Float16, kProjGated, false, false>(p, groups, s);
  if (mode == kProjSum) return launch_projection_small<_Float16, kProjSum, false, true>(p, groups, s);
  return launch_projection_small<_Float16, kProjPlain, true, true>(p, groups, s);
}
}  // namespace cmpext3
