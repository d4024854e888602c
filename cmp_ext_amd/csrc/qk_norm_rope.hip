// Norms of queries and keys for each head with the position rotation, in one pass over both:
//   y = x * rsqrt(mean(x^2) + eps) * weight,  pairs (a, b) -> (a cos - b sin, b cos + a sin).
// Bound by reading and writing every element once: 8192 tokens of 40 heads of 128 in 37 us on MI355X,
// 4.7 TB/s (a large copy moves 5.25), in fp32 71.5; a few tokens by the launch, 4 us, and the call from the host, 5.
//
// Vector kernel (rows of 16-byte pieces): a head belongs to dim / 16 neighbouring lanes (rounded
// up to a power of two), and a lane holds the two pieces of 8 elements whose elements pair up
// (half layout: pieces i and rotary / 16 + i; neighbouring pairs: pieces 2i and 2i + 1), so
// that only the sum of squares crosses lanes.  (Two or four heads a lane, with one row of the tables:
// no faster.)  The tables are read as fp32, one row per token,
// shared by its heads through the caches.
// General kernel (any dim, alignment): one wave per head, an element at a time, its partner read again: 200 us
// for those tokens with heads of 100 (26 for their bytes at the copy's rate).
#include "attention_params.h"
#include "device_common.h"

namespace cmpext3 {

// Eight elements of a row as floats, and back (rounded to nearest even).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
    const u32x4 v = *(const u32x4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = from_bits<T>((uint16_t)v[i]);
      x[2 * i + 1] = from_bits<T>((uint16_t)(v[i] >> 16));
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
    *(f32x4*)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    // streamed past the caches' reusable lines (8192 tokens of 40 heads of 128: 40.9 -> 36.3 us)
    __builtin_nontemporal_store(u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])},
                                (u32x4*)p);
  }
}

// LANES: lanes of a head, a power of two.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) qk_norm_rope_vec_kernel(const RopeParams p) {
  const int per_token = p.heads[0] + p.heads[1];
  const int64_t unit = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int i = threadIdx.x % LANES;
  const int64_t token = unit / per_token;
  int head = (int)(unit - token * per_token);
  const int which = head >= p.heads[0];
  if (which) head -= p.heads[0];
  const bool live = token < p.tokens && 16 * i < p.dim;
  // the lane's two pieces, and whether they turn
  const int pairs = p.rotary / 16;  // lanes that turn
  const bool turn = i < pairs;
  int e0, e1;
  if (p.interleaved || !turn) {
    e0 = 16 * i;
    e1 = e0 + 8;
  } else {
    e0 = 8 * i;
    e1 = p.rotary / 2 + 8 * i;
  }
  float x[16];
  float c[8], s[8];
  if (live) {
    const T* row = (const T*)p.x[which] + token * p.x_token[which] + head * p.x_head[which];
    load8(row + e0, x);
    load8(row + e1, x + 8);
    if (turn) {
      const int64_t pos = p.positions[token];
      if ((uint64_t)pos < (uint64_t)p.table_rows) {
        load8(p.cos + pos * p.table_row + 8 * i, c);
        load8(p.sin + pos * p.table_row + 8 * i, s);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = s[j] = __builtin_nanf("");
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = 0.f;
  }
  if (p.weight[which] != nullptr) {
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) sq = __builtin_fmaf(x[j], x[j], sq);
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) sq += __shfl_xor(sq, m);
    const float r = 1.0f / __builtin_sqrtf(sq / (float)p.dim + p.eps);
    float w[16];
    if (live) {
      load8((const T*)p.weight[which] + e0, w);
      load8((const T*)p.weight[which] + e1, w + 8);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] *= r * w[j];
    }
  }
  if (!live) return;
  if (turn) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int a = p.interleaved ? 2 * j : j, b = p.interleaved ? 2 * j + 1 : 8 + j;
      const float u = x[a], v = x[b];
      x[a] = u * c[j] - v * s[j];
      x[b] = v * c[j] + u * s[j];
    }
  }
  T* out = (T*)p.y[which] + token * p.y_token[which] + head * p.y_head[which];
  store8(out + e0, x);
  store8(out + e1, x + 8);
}

template <typename T>
__device__ __forceinline__ float load1(const T* p) { return (float)*p; }

// One wave per head.  A row may be its own output: all of it is read before any is written.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_any_kernel(const RopeParams p) {
  constexpr int kMost = 16;  // elements of a lane: dim <= 1024
  const int lane = threadIdx.x & 63;
  const int per_token = p.heads[0] + p.heads[1];
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t token = unit / per_token;
  if (token >= p.tokens) return;
  int head = (int)(unit - token * per_token);
  const int which = head >= p.heads[0];
  if (which) head -= p.heads[0];
  const T* row = (const T*)p.x[which] + token * p.x_token[which] + head * p.x_head[which];
  const T* weight = (const T*)p.weight[which];
  float x[kMost];
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int e = 64 * k + lane;
    x[k] = e < p.dim ? load1(row + e) : 0.f;
    sq = __builtin_fmaf(x[k], x[k], sq);
  }
  float r = 1.f;
  if (weight != nullptr) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) sq += __shfl_xor(sq, m);
    r = 1.0f / __builtin_sqrtf(sq / (float)p.dim + p.eps);
  }
  const int64_t pos = p.positions[token];
  const bool known = (uint64_t)pos < (uint64_t)p.table_rows;
  const int half = p.rotary / 2;
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int e = 64 * k + lane;
    if (e >= p.dim) continue;
    float y = weight != nullptr ? x[k] * (r * load1(weight + e)) : x[k];
    if (e < p.rotary) {
      const bool second = p.interleaved ? e & 1 : e >= half;
      const int f = p.interleaved ? e ^ 1 : second ? e - half : e + half;
      const int n = p.interleaved ? e >> 1 : second ? e - half : e;
      float z = load1(row + f);
      if (weight != nullptr) z *= r * load1(weight + f);
      const float c = known ? p.cos[pos * p.table_row + n] : __builtin_nanf("");
      const float s = known ? p.sin[pos * p.table_row + n] : __builtin_nanf("");
      y = second ? y * c + z * s : y * c - z * s;
    }
    x[k] = y;
  }
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // the whole row is read
  T* out = (T*)p.y[which] + token * p.y_token[which] + head * p.y_head[which];
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int e = 64 * k + lane;
    if (e < p.dim) out[e] = (T)x[k];
  }
}

template <typename T>
static hipError_t launch_rope(bool vec, const RopeParams& p, hipStream_t s) {
  const int64_t units = p.tokens * (p.heads[0] + p.heads[1]);
  if (!vec) return launch_kernel(qk_norm_rope_any_kernel<T>, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, p);
  const int lanes = p.dim <= 64 ? 4 : p.dim <= 128 ? 8 : p.dim <= 256 ? 16 : p.dim <= 512 ? 32 : 64;
  const dim3 grid((unsigned)((units * lanes + 255) / 256)), block(256);
  switch (lanes) {
    case 4: return launch_kernel(qk_norm_rope_vec_kernel<T, 4>, grid, block, 0, s, p);
    case 8: return launch_kernel(qk_norm_rope_vec_kernel<T, 8>, grid, block, 0, s, p);
    case 16: return launch_kernel(qk_norm_rope_vec_kernel<T, 16>, grid, block, 0, s, p);
    case 32: return launch_kernel(qk_norm_rope_vec_kernel<T, 32>, grid, block, 0, s, p);
    default: return launch_kernel(qk_norm_rope_vec_kernel<T, 64>, grid, block, 0, s, p);
  }
}

hipError_t launch_qk_norm_rope(int dtype, bool vec, const RopeParams& p, hipStream_t s) {
  return dtype == kF16 ? launch_rope<_Float16>(vec, p, s)
         : dtype == kBF16 ? launch_rope<__bf16>(vec, p, s) : launch_rope<float>(vec, p, s);
}

}  // namespace cmpext3
