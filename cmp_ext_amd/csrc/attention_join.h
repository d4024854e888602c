// Ranges of keys ("splits") that attention kernels sum apart, and joining them: with
// m = max m_s over a row's splits (a row: one query of one head),
//   out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s,
// always in the order of the splits.  The workgroups of one row tile leave their sums in one
// stretch of the workspace, [split][rows * dim of O, then rows of (m, l)], as device-coherent
// stores.  The last of them to finish joins them (counted in by split_counters, zero again
// afterwards), where the stream has counters; else a second launch does.  Bound by the bytes of the
// sums, out and back, and by the last workgroup's latency: about 5 of 126 us on MI355X for the splits of
// 224 tiles of 128 rows of 128.
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
__device__ __forceinline__ int splits_of(const AttnParams& p, const Seq& s, int end) {
  return p.splits == 1 ? 1 : min(p.splits, max(1, (end + s.split_keys - 1) / s.split_keys));
}

// IT items (four elements of a row) of each thread, SP splits of each at a time: so many loads on
// their way.  `share` threads take the splits of an item in turn (share > 1: all items at once).
template <typename T, int IT, int SP, int THREADS>
__device__ __forceinline__ void join_items(const AttnParams& p, const Seq& sq, int kvh, int row0, int rows, const float* part, int bm, int n,
                                           int share, const float* weight, const float* inv, f32x4* sums) {
  const int tid = threadIdx.x, quads = p.dim / 4, items = rows * quads;
  const int mine = share > 1 ? tid / items : 0;
  for (int i0 = 0; i0 < items; i0 += THREADS * IT) {
    f32x4 acc[IT];
    int r[IT], e[IT];
    bool busy[IT];
#pragma unroll
    for (int t = 0; t < IT; ++t) {
      const int i = share > 1 ? tid - mine * items : i0 + t * THREADS + tid;
      busy[t] = i < items && mine < share;
      r[t] = busy[t] ? i / quads : 0;
      e[t] = busy[t] ? 4 * (i - r[t] * quads) : 0;
      acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int s0 = mine; s0 < n; s0 += SP * share) {
      f32x4 x[IT][SP];
      float w[IT][SP];
      // past the last split the last one again: no load waits behind a branch.  It is its sum that is made
      // zero, not its weight, which would make NaN of an infinite one.
#pragma unroll
      for (int t = 0; t < IT; ++t)
#pragma unroll
        for (int j = 0; j < SP; ++j)
          x[t][j] = load16_coherent(part, part_at(p, bm, min(s0 + j * share, n - 1)) + part_o(p, r[t]) + 4 * e[t]);
#pragma unroll
      for (int t = 0; t < IT; ++t)
#pragma unroll
        for (int j = 0; j < SP; ++j) w[t][j] = weight[r[t] * n + min(s0 + j * share, n - 1)];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < IT; ++t)
#pragma unroll
        for (int j = 0; j < SP; ++j) acc[t] += w[t][j] * (s0 + j * share < n ? x[t][j] : f32x4{0.f, 0.f, 0.f, 0.f});
    }
    if (share > 1) {  // uniform
      sums[tid] = acc[0];
      __syncthreads();
      if (busy[0] && mine == 0)
        for (int g = 1; g < share; ++g) acc[0] += sums[tid + g * items];
    }
#pragma unroll
    for (int t = 0; t < IT; ++t) {
      if (!busy[t] || mine != 0) continue;
      const int row = row0 + r[t], tok = row / p.group, head = kvh * p.group + row - tok * p.group;
      T* op = (T*)p.out + sq.b * p.out_batch + (int64_t)(sq.q0 + tok) * p.out_token + (int64_t)head * p.out_head;
      const float f = inv[r[t]];
      *(u32x2*)(op + e[t]) = u32x2{round2<T>(acc[t][0] * f, acc[t][1] * f), round2<T>(acc[t][2] * f, acc[t][3] * f)};
    }
  }
}

// Joins n > 1 splits of a tile's `rows` rows (of room for bm) and writes them out.  The workgroup's
// THREADS threads, all of them here, with 16 THREADS + 4 bm (n + 1) bytes of LDS.
template <typename T, int THREADS>
__device__ __forceinline__ void join_rows(const AttnParams& p, const Seq& sq, int kvh, int row0, int rows, const float* part, int bm,
                                          int n, unsigned char* lds) {
  const int tid = threadIdx.x;
  f32x4* sums = (f32x4*)lds;
  float* inv = (float*)(sums + THREADS);  // 1 / the rows' sums
  float* weight = inv + bm;           // [row][split]: 2^(m_s - m)
  // the lanes of a row, a power of two up to a wave: 256 threads at most
  const int lanes = rows <= 4 ? 64 : rows <= 8 ? 32 : rows <= 16 ? 16 : rows <= 32 ? 8 : rows <= 64 ? 4 : 2;
  const int r = tid / lanes;
  float m = -INFINITY, l = 0.f;
  if (r < rows)
    for (int s = tid % lanes; s < n; s += lanes) {
      const float x = __uint_as_float(load8_coherent(part, part_at(p, bm, s) + part_ml(p, bm, r)).x);
      weight[r * n + s] = x;
      m = fmaxf(m, x);
    }
  for (int x = 1; x < lanes; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
  if (r < rows)
    for (int s = tid % lanes; s < n; s += lanes) {
      const float f = m == -INFINITY ? 0.f : exp2_hw(weight[r * n + s] - m);
      weight[r * n + s] = f;
      l += f * __uint_as_float(load8_coherent(part, part_at(p, bm, s) + part_ml(p, bm, r)).y);
    }
  for (int x = 1; x < lanes; x <<= 1) l += __shfl_xor(l, x);
  if (r < rows && tid % lanes == 0) inv[r] = row_factor(p, sq, row0 + r, l);
  __syncthreads();
  const int items = rows * (p.dim / 4);
  if (items <= THREADS / 2)
    join_items<T, 1, 16, THREADS>(p, sq, kvh, row0, rows, part, bm, n, THREADS / items, weight, inv, sums);
  else
    join_items<T, 4, 4, THREADS>(p, sq, kvh, row0, rows, part, bm, n, 1, weight, inv, sums);
}

// After a workgroup has stored its split: joins, if it is the last of its tile's n.
template <typename T, int THREADS>
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
  join_rows<T, THREADS>(p, sq, kvh, row0, rows, part, bm, n, lds);
  if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next kernel
}

// The stretch of a workgroup's row tile.
__device__ __forceinline__ float* part_of_tile(const AttnParams& p, int bm) {
  return p.part + (int64_t)blockIdx.x * p.splits * bm * (p.dim + 2);
}

}  // namespace cmpext3
