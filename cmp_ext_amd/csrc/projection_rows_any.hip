// Kernels for few rows of x, weights of any alignment: every element type and mode.
#include "projection_rows_any_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_rows_any(int dtype, ProjMode mode, const ProjParams& p, hipStream_t s) {
  if (dtype == kF16) return launch_projection_rows_any<_Float16, kProjGated>(p, s);
  if (dtype == kBF16) return launch_projection_rows_any<__bf16, kProjGated>(p, s);
  if (mode == kProjGated) return launch_projection_rows_any<int8_t, kProjGated>(p, s);
  return launch_projection_rows_any<int8_t, kProjPlain>(p, s);
}
}  // namespace cmpext3
