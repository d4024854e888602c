#include "attention_few_kernel.h"

namespace cmpext3 {
hipError_t launch_attention_few_bf16_paged8(int hd, int blocks16, int waves, const AttnParams& p, dim3 grid, hipStream_t s) {
  return blocks16 == 1 ? launch_few_hd<__bf16, kKvPaged8, 1>(hd, waves, p, grid, s) : launch_few_hd<__bf16, kKvPaged8, 2>(hd, waves, p, grid, s);
}
}  // namespace cmpext3
