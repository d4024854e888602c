#include "attention_few_kernel.h"

namespace cmpext3 {
hipError_t launch_attention_few_f16_paged16(int hd, int blocks16, int waves, const AttnParams& p, dim3 grid, hipStream_t s) {
  return blocks16 == 1 ? launch_few_hd<_Float16, kKvPaged16, 1>(hd, waves, p, grid, s) : launch_few_hd<_Float16, kKvPaged16, 2>(hd, waves, p, grid, s);
}
}  // namespace cmpext3
