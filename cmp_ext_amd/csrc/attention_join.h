// Ranges of keys ("splits") that attention kernels sum apart, and joining them: with
// m = max m_s over a row's splits (a row: one query of one head),
//   out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s,
// always in the order of the splits.  The workgroups of one row tile leave their sums in one
// stretch of the workspace, [split][rows * dim of O, then rows of (m, l)], as device-coherent
// stores.  The last of them to finish joins them (counted in by split_counters, zero again
// afterwards), where the stream has counters; else a second launch does.
#pragma once

#include "attention_common.h"

namespace cmpext3 {

__device__ __forceinline__ void store8_coherent(float* base, uint32_t off, float x, float y) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, (int)kBufRecords, kBufWord3);
  __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(x), __float_as_uint(y)}, r, off, 0, kCoherent);
}
__device__ __forceinline__ u32x2 load8_coherent(const float* base, uint32_t off) {
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, (int)kBufRecords, kBufWord3);
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, kCoherent));
}

// Bytes from a tile's stretch to its split s, and from there to row r's O and to its (m, l).
__device__ __forceinline__ uint32_t part_at(const AttnParams& p, int bm, int s) { return (uint32_t)(s * bm * (p.dim + 2)) * 4u; }
__device__ __forceinline__ uint32_t part_o(const AttnParams& p, int r) { return (uint32_t)(r * p.dim) * 4u; }
__device__ __forceinline__ uint32_t part_ml(const AttnParams& p, int bm, int r) { return (uint32_t)(bm * p.dim + 2 * r) * 4u; }

// Splits that a row tile has: those that hold a key before `end`, at least one.
__device__ __forceinline__ int splits_of(const AttnParams& p, int end) {
  return p.splits == 1 ? 1 : min(p.splits, max(1, (end + p.split_keys - 1) / p.split_keys));
}

// Joins n > 1 splits of a tile's `rows` rows (of room for bm) and writes them out.  256 threads,
// all of them here, with 8 * bm * n bytes of LDS (at least 4 KB).
template <typename T>
__device__ __forceinline__ void join_rows(const AttnParams& p, const Seq& sq, int kvh, int row0, int rows, const float* part, int bm,
                                          int n, unsigned char* lds) {
  const int tid = threadIdx.x;
  u32x2* ml = (u32x2*)lds;  // [row][split]
  for (int i = tid; i < rows * n; i += 256) {
    const int r = i / n, s = i - r * n;
    ml[i] = load8_coherent(part, part_at(p, bm, s) + part_ml(p, bm, r));
  }
  __syncthreads();
  const int quads = p.dim / 4, items = rows * quads;  // an item: four elements of a row
  // where the items are few, several threads take an item's splits in turn
  const int share = max(1, 256 / items), mine = share > 1 ? tid / items : 0;
  for (int i0 = 0; i0 < items; i0 += 256) {
    const int i = share > 1 ? tid - mine * items : i0 + tid;
    const bool busy = i < items && mine < share;
    const int r = busy ? i / quads : 0, e = 4 * (i - r * quads);
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    if (busy) {
      float m = -INFINITY;
      for (int s = 0; s < n; ++s) m = fmaxf(m, __uint_as_float(ml[r * n + s].x));
      if (m != -INFINITY) {
        for (int s0 = mine; s0 < n; s0 += 8 * share) {
          f32x4 x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (s0 + j * share < n) x[j] = load16_coherent(part, part_at(p, bm, s0 + j * share) + part_o(p, r) + 4 * e);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (s0 + j * share < n) {
              const u32x2 v = ml[r * n + s0 + j * share];
              const float f = exp2_hw(__uint_as_float(v.x) - m);
              l += f * __uint_as_float(v.y);
              acc += f * x[j];
            }
        }
      }
    }
    if (share > 1) {  // uniform; items <= 128 here, one turn
      __syncthreads();
      f32x4* sums = (f32x4*)lds;
      float* ls = (float*)(sums + 256);
      sums[tid] = acc;
      ls[tid] = l;
      __syncthreads();
      if (!busy || mine != 0) continue;
      for (int g = 1; g < share; ++g) {
        acc += sums[tid + g * items];
        l += ls[tid + g * items];
      }
    }
    if (!busy) continue;
    const int row = row0 + r, tok = row / p.group, head = kvh * p.group + row - tok * p.group;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    T* op = (T*)p.out + sq.b * p.out_batch + (int64_t)(sq.q0 + tok) * p.out_token + (int64_t)head * p.out_head;
    *(u32x2*)(op + e) = u32x2{round2<T>(acc[0] * inv, acc[1] * inv), round2<T>(acc[2] * inv, acc[3] * inv)};
  }
}

// After a workgroup has stored its split: joins, if it is the last of its tile's n.
template <typename T>
__device__ __forceinline__ void join_if_last(const AttnParams& p, const Seq& sq, int kvh, int row0, int rows, const float* part, int bm,
                                             int n, unsigned char* lds) {
  if (p.sem == nullptr) return;
  __shared__ int last;
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // this wave's stores are done
  __syncthreads();
  unsigned int* count = p.sem + blockIdx.x;
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(n - 1);
  __syncthreads();
  if (!last) return;
  join_rows<T>(p, sq, kvh, row0, rows, part, bm, n, lds);
  if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next kernel
}

// The stretch of a workgroup's row tile.
__device__ __forceinline__ float* part_of_tile(const AttnParams& p, int bm) {
  return p.part + (int64_t)blockIdx.x * p.splits * bm * (p.dim + 2);
}

}  // namespace cmpext3
