// The second launch that joins splits of the keys where the kernel that summed them had no
// counters (attention_join.h): one workgroup per row tile.
#include "attention_join.h"

namespace cmpext3 {

template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams p, int bm) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[kJoinBytes];
  const int kvh = blockIdx.x % p.kv_heads;
  const Seq sq = seq_of_slot<true>(p, blockIdx.x / p.kv_heads, bm);
  if (sq.b < 0) return;
  const int row0 = sq.tile * bm, rows = min(bm, sq.len_q * p.group - row0);
  const int n = splits_of(p, sq, keys_end(p, sq, row0 + rows - 1));
  if (n > 1) join_rows<T, 256>(p, sq, kvh, row0, rows, part_of_tile(p, bm), bm, n, lds);
}

hipError_t launch_attention_join(int dtype, int bm, const AttnParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.slots * p.kv_heads)), block(256);
  return dtype == kF16 ? launch_kernel(attention_join_kernel<_Float16>, grid, block, 0, s, p, bm)
                       : launch_kernel(attention_join_kernel<__bf16>, grid, block, 0, s, p, bm);
}

}  // namespace cmpext3
