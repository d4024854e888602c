// Joins the ranges of keys ("splits") that attention kernels summed apart: with
// m = max m_s over a row's splits,
//   out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.
// One workgroup per row (a query of a head); wave w takes splits w, w + 4, ..., each lane four
// consecutive elements of the head (two groups of elements beside each other where the head
// has at most 128), and the waves meet in LDS.
#include "attention_common.h"

namespace cmpext3 {

constexpr int kJoinWaves = 4;

template <typename T>
__global__ void __launch_bounds__(64 * kJoinWaves) attention_join_kernel(const AttnParams p) {
  __shared__ float part[kJoinWaves][256 + 4];
  __shared__ float part_l[kJoinWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const int token = (int)(row / p.heads), head = (int)(row - (int64_t)token * p.heads);
  // the row's sequence and its number of keys
  int b, len_k, local;
  if (p.starts_q == nullptr) {
    b = token / p.len_q;
    local = token - b * p.len_q;
  } else {
    int count = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
      const unsigned long long m =
          __builtin_amdgcn_ballot_w64(b0 + lane < p.batch && clampi(p.starts_q[min(b0 + lane, p.batch - 1)], 0, p.total_q) <= token);
      count += __builtin_popcountll(m);
      if (m != ~0ull) break;
    }
    b = count - 1;
    if (b < 0 || token >= clampi(p.starts_q[b + 1], 0, p.total_q)) return;  // in no sequence
    local = token;
  }
  if (p.kv.table != nullptr) {
    len_k = (int)min((int64_t)max(p.seq_lens[b], 0), (int64_t)p.kv.table_pages * p.kv.page_size);
  } else if (p.starts_k != nullptr) {
    const int k0 = clampi(p.starts_k[b], 0, p.total_k);
    len_k = clampi(p.starts_k[b + 1], k0, p.total_k) - k0;
  } else {
    len_k = p.len_k;
  }
  const int n = max(1, (len_k + p.split_keys - 1) / p.split_keys);  // its splits: the grid has no fewer
  float m = -INFINITY;
  for (int s = lane; s < n; s += 64) m = fmaxf(m, p.part_ml[2 * ((int64_t)s * p.rows + row)]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  if (m != -INFINITY) {
#pragma unroll 4
    for (int s = wave; s < n; s += kJoinWaves) {
      const int64_t at = (int64_t)s * p.rows + row;
      const float f = exp2_hw(p.part_ml[2 * at] - m);
      l += f * p.part_ml[2 * at + 1];
      if (4 * lane < p.dim) acc += f * *(const f32x4*)(p.part_o + at * p.dim + 4 * lane);
    }
  }
  *(f32x4*)&part[wave][4 * lane] = acc;
  if (lane == 0) part_l[wave] = l;
  __syncthreads();
  if (wave != 0 || 4 * lane >= p.dim) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) {
    acc += *(const f32x4*)&part[w][4 * lane];
    l += part_l[w];
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  T* op = (T*)p.out + (int64_t)(p.starts_q ? 0 : b) * p.out_batch + (int64_t)local * p.out_token + (int64_t)head * p.out_head;
  *(u32x2*)(op + 4 * lane) = u32x2{pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv)};
}

hipError_t launch_attention_join(int dtype, const AttnParams& p, hipStream_t s) {
  const dim3 grid((unsigned)p.rows), block(64 * kJoinWaves);
  return dtype == 0 ? launch_kernel(attention_join_kernel<_Float16>, grid, block, 0, s, p)
                    : launch_kernel(attention_join_kernel<__bf16>, grid, block, 0, s, p);
}

}  // namespace cmpext3
