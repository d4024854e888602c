// Kernels for few rows of x, weights of whole 16 bytes a row: every element type and mode.
#include "projection_rows_kernel.h"

namespace cmpext3 {
hipError_t launch_projection_rows(int dtype, ProjMode mode, const ProjParams& p, hipStream_t s) {
  if (dtype == kF16) return launch_projection_rows<_Float16, kProjGated>(p, s);
  if (dtype == kBF16) return launch_projection_rows<__bf16, kProjGated>(p, s);
  if (mode == kProjGated) return launch_projection_rows<int8_t, kProjGated>(p, s);
  return launch_projection_rows<int8_t, kProjPlain>(p, s);
}
hipError_t launch_projection_rows_codes(int x_dtype, ProjMode mode, const ProjParams& p, hipStream_t s) {
  if (x_dtype == kF16)
    return mode == kProjGated ? launch_projection_rows_codes<_Float16, kProjGated>(p, s) : launch_projection_rows_codes<_Float16, kProjPlain>(p, s);
  return mode == kProjGated ? launch_projection_rows_codes<__bf16, kProjGated>(p, s) : launch_projection_rows_codes<__bf16, kProjPlain>(p, s);
}
}  // namespace cmpext3
