// Writing keys and values into a paged cache, in 16 bits or as e4m3 codes with a scale for each
// token and head, and reading sequences back as packed rows.  Both are bound by the bytes they
// move (launch latency for a few tokens).
//
// Codes: with a = max(max |x|, 2^-100) over the row's finite elements,
//   code = e4m3(x * (448 / a)),  scale = a / 448:
// the largest element becomes the largest code, and 2^-100 keeps both quotients ordinary floats.
// The divisions are correctly rounded, once per row.  An element that is not finite becomes NaN
// by itself and leaves the row's scale alone.
#include "attention_common.h"

namespace cmpext3 {

constexpr float kE4m3Most = 448.f;
constexpr float kLeastAmax = 0x1p-100f;

// Rows of 8 elements per lane: LANES neighbouring lanes (a power of two, at least dim / 8).
// grid: rows of keys, then rows of values.
template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256) kv_cache_write_kernel(const CacheParams p) {
  const int64_t rows = p.tokens * p.kv_heads;
  int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int e = 8 * (threadIdx.x % LANES);
  const bool value = row >= rows;
  if (value) row -= rows;
  const int64_t token = row / p.kv_heads;
  const int head = (int)(row - token * p.kv_heads);
  const bool live = token < p.tokens && e < p.dim;
  u32x4 x = u32x4{0, 0, 0, 0};
  int64_t slot = -1;
  if (live) {
    slot = p.slots[token];
    const T* in = value ? (const T*)p.v_in + token * p.v_in_token + head * p.v_in_head
                        : (const T*)p.k_in + token * p.k_in_token + head * p.k_in_head;
    x = *(const u32x4*)(in + e);
  }
  const bool kept = live && (uint64_t)slot < (uint64_t)p.kv.pages * (uint64_t)p.kv.page_size;
  const int64_t page = kept ? slot / p.kv.page_size : 0, place = kept ? slot - page * p.kv.page_size : 0;
  const int64_t at = value ? page * p.kv.v_page + place * p.kv.v_token + head * p.kv.v_head
                           : page * p.kv.k_page + place * p.kv.k_token + head * p.kv.k_head;
  void* cache = const_cast<void*>(value ? p.kv.v : p.kv.k);
  if constexpr (!E4M3) {
    if (kept) *(u32x4*)((T*)cache + at + e) = x;
  } else {
    float f[8];
    float a = kLeastAmax;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = from_bits<T>((uint16_t)x[i]);
      f[2 * i + 1] = from_bits<T>((uint16_t)(x[i] >> 16));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!__builtin_isfinite(f[i])) f[i] = __builtin_nanf("");
      a = fmaxf(a, fabsf(f[i]));  // fmaxf passes over NaN
    }
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) a = fmaxf(a, __shfl_xor(a, m));
    if (!kept) return;
    const float inv = kE4m3Most / a;
    uint32_t code[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = f[4 * h + i] * inv;
        // the product may round to just above 448; NaN stays
        y[i] = y[i] > kE4m3Most ? kE4m3Most : y[i] < -kE4m3Most ? -kE4m3Most : y[i];
      }
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
      code[h] = (uint32_t)c;
    }
    *(u32x2*)((uint8_t*)cache + at + e) = u32x2{code[0], code[1]};
    if (e == 0) {
      float* scale = const_cast<float*>(value ? p.kv.v_scale : p.kv.k_scale);
      scale[value ? page * p.kv.vs_page + place * p.kv.vs_token + head * p.kv.vs_head
                  : page * p.kv.ks_page + place * p.kv.ks_token + head * p.kv.ks_head] = a / kE4m3Most;
    }
  }
}

template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256) kv_cache_read_kernel(const CacheParams p) {
  const int64_t rows = p.tokens * p.kv_heads;
  int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int e = 8 * (threadIdx.x % LANES);
  const bool value = row >= rows;
  if (value) row -= rows;
  const int64_t token = row / p.kv_heads;
  const int head = (int)(row - token * p.kv_heads);
  if (token >= p.tokens || e >= p.dim) return;
  // the last sequence that starts at or before the row
  int lo = 0, hi = p.batch;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.starts[mid] <= token) lo = mid + 1;
    else hi = mid;
  }
  const int b = lo - 1;
  u32x4 x = u32x4{0, 0, 0, 0};
  if (b >= 0 && token < p.starts[b + 1]) {
    const int64_t key = token - p.starts[b];
    if (key < (int64_t)p.kv.table_pages * p.kv.page_size) {
      int place;
      const int page = page_of(p.kv, p.kv.table + b * p.kv.table_row, (int)key, place);
      if (page >= 0) {
        const int64_t at = value ? page * p.kv.v_page + place * p.kv.v_token + head * p.kv.v_head
                                 : page * p.kv.k_page + place * p.kv.k_token + head * p.kv.k_head;
        const void* cache = value ? p.kv.v : p.kv.k;
        if constexpr (!E4M3) {
          x = *(const u32x4*)((const T*)cache + at + e);
        } else {
          const float s = value ? p.kv.v_scale[page * p.kv.vs_page + place * p.kv.vs_token + head * p.kv.vs_head]
                                : p.kv.k_scale[page * p.kv.ks_page + place * p.kv.ks_token + head * p.kv.ks_head];
          const u32x2 c = *(const u32x2*)((const uint8_t*)cache + at + e);
          typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f32x2 u = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false), v = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
            float y[4] = {u[0] * s, u[1] * s, v[0] * s, v[1] * s};
            // the value is the fp32 product, rounded to 32 bits before 16: kept from being taken
            // as one mixed-precision instruction, which rounds once
#pragma unroll
            for (int i = 0; i < 4; ++i) asm("" : "+v"(y[i]));
            x[2 * h] = pack2<T>(y[0], y[1]);
            x[2 * h + 1] = pack2<T>(y[2], y[3]);
          }
        }
      }
    }
  }
  *(u32x4*)((T*)(value ? p.v_out : p.k_out) + row * p.dim + e) = x;
}

template <typename T, bool E4M3, bool WRITE>
static hipError_t launch_cache(const CacheParams& p, hipStream_t s) {
  const int lanes = p.dim <= 64 ? 8 : p.dim <= 128 ? 16 : 32;
  const dim3 grid((unsigned)((2 * p.tokens * p.kv_heads * lanes + 255) / 256)), block(256);
  if constexpr (WRITE) {
    if (lanes == 8) return launch_kernel(kv_cache_write_kernel<T, E4M3, 8>, grid, block, 0, s, p);
    if (lanes == 16) return launch_kernel(kv_cache_write_kernel<T, E4M3, 16>, grid, block, 0, s, p);
    return launch_kernel(kv_cache_write_kernel<T, E4M3, 32>, grid, block, 0, s, p);
  } else {
    if (lanes == 8) return launch_kernel(kv_cache_read_kernel<T, E4M3, 8>, grid, block, 0, s, p);
    if (lanes == 16) return launch_kernel(kv_cache_read_kernel<T, E4M3, 16>, grid, block, 0, s, p);
    return launch_kernel(kv_cache_read_kernel<T, E4M3, 32>, grid, block, 0, s, p);
  }
}

hipError_t launch_kv_cache_write(int dtype, bool e4m3, const CacheParams& p, hipStream_t s) {
  if (dtype == kF16) return e4m3 ? launch_cache<_Float16, true, true>(p, s) : launch_cache<_Float16, false, true>(p, s);
  return e4m3 ? launch_cache<__bf16, true, true>(p, s) : launch_cache<__bf16, false, true>(p, s);
}
hipError_t launch_kv_cache_read(int dtype, bool e4m3, const CacheParams& p, hipStream_t s) {
  if (dtype == kF16) return e4m3 ? launch_cache<_Float16, true, false>(p, s) : launch_cache<_Float16, false, false>(p, s);
  return e4m3 ? launch_cache<__bf16, true, false>(p, s) : launch_cache<__bf16, false, false>(p, s);
}

}  // namespace cmpext3
