#include "attention_tile_kernel.h"

namespace cmpext3 {
hipError_t launch_attention_tile_bf16_paged8(int hd, int ks, const AttnParams& p, dim3 grid, hipStream_t s) {
  return launch_tile_hd<__bf16, kKvPaged8>(hd, ks, p, grid, s);
}
}  // namespace cmpext3
