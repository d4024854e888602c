// Writing keys and values into a paged cache, in 16 bits or as e4m3 codes with a scale for each
// token and head, and reading sequences back as packed rows.  Both are bound by the bytes they
// move (MI355X, 8 heads of 128 as codes: 31469 tokens read back, 193 MB, in 38 us, 5.1 TB/s, as a large
// copy), a few tokens by the launch (16 written 4 us, 1064 written 5).
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

// Eight elements of a row as the cache holds them.  The lanes of a row (LANES, a power of two) share
// its largest element.
template <typename T, int LANES>
__device__ __forceinline__ u32x2 codes_of(u32x4 x, float& scale) {
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
  const float inv = kE4m3Most / a;
  scale = a / kE4m3Most;
  u32x2 code;
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
  return code;
}

// Eight elements of a key's row and of its value's per lane, LANES neighbouring lanes to a row (at
// least dim / 8).
template <typename T, bool E4M3, int LANES>
__global__ void __launch_bounds__(256) kv_cache_write_kernel(const CacheParams p) {
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int e = 8 * (threadIdx.x % LANES);
  const int64_t token = row / p.kv_heads;
  const int head = (int)(row - token * p.kv_heads);
  const bool live = token < p.tokens && e < p.dim;
  u32x4 k = u32x4{0, 0, 0, 0}, v = u32x4{0, 0, 0, 0};
  int64_t slot = -1;
  if (live) {
    slot = p.slots[token];
    k = *(const u32x4*)((const T*)p.k_in + token * p.k_in_token + head * p.k_in_head + e);
    v = *(const u32x4*)((const T*)p.v_in + token * p.v_in_token + head * p.v_in_head + e);
  }
  const bool kept = live && (uint64_t)slot < (uint64_t)p.kv.pages * (uint64_t)p.kv.page_size;
  int64_t page = 0, place = 0;
  if (kept) {
    page = p.kv.page_shift >= 0 ? slot >> p.kv.page_shift : slot / p.kv.page_size;
    place = slot - page * p.kv.page_size;
  }
  const int64_t k_at = page * p.kv.k_page + place * p.kv.k_token + head * p.kv.k_head + e;
  const int64_t v_at = page * p.kv.v_page + place * p.kv.v_token + head * p.kv.v_head + e;
  if constexpr (!E4M3) {
    if (!kept) return;
    *(u32x4*)((T*)const_cast<void*>(p.kv.k) + k_at) = k;
    *(u32x4*)((T*)const_cast<void*>(p.kv.v) + v_at) = v;
  } else {
    float ks, vs;
    const u32x2 kc = codes_of<T, LANES>(k, ks), vc = codes_of<T, LANES>(v, vs);
    if (!kept) return;
    *(u32x2*)((uint8_t*)const_cast<void*>(p.kv.k) + k_at) = kc;
    *(u32x2*)((uint8_t*)const_cast<void*>(p.kv.v) + v_at) = vc;
    if (e == 0) {
      const_cast<float*>(p.kv.k_scale)[page * p.kv.ks_page + place * p.kv.ks_token + head * p.kv.ks_head] = ks;
      const_cast<float*>(p.kv.v_scale)[page * p.kv.vs_page + place * p.kv.vs_token + head * p.kv.vs_head] = vs;
    }
  }
}

// EPL elements of a row from the cache, as EPL / 8 pieces of T.
template <typename T, bool E4M3, int EPL>
__device__ __forceinline__ void read_row(const void* cache, int64_t at, float s, u32x4* x) {
  if constexpr (!E4M3) {
    x[0] = *(const u32x4*)((const T*)cache + at);
  } else {
    uint32_t c[EPL / 4];
    if constexpr (EPL == 16) {
      const u32x4 v = __builtin_nontemporal_load((const u32x4_a8*)((const uint8_t*)cache + at));
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = v[i];
    } else {
      const u32x2 v = *(const u32x2*)((const uint8_t*)cache + at);
      c[0] = v.x, c[1] = v.y;
    }
    typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int h = 0; h < EPL / 4; ++h) {
      const f32x2 u = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false), v = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
      float y[4] = {u[0] * s, u[1] * s, v[0] * s, v[1] * s};
      // the value is the fp32 product, rounded to 32 bits before 16: kept from being taken
      // as one mixed-precision instruction, which rounds once
#pragma unroll
      for (int i = 0; i < 4; ++i) asm("" : "+v"(y[i]));
      x[h / 2][2 * (h & 1)] = round2<T>(y[0], y[1]);
      x[h / 2][2 * (h & 1) + 1] = round2<T>(y[2], y[3]);
    }
  }
}

// A thread takes EPL elements of a key's row and of its value's: the sequence, page and place are
// found once for both.  (31469 tokens of 8 heads of 128, the write of 1064 of them included: 43.6 us
// on MI355X; with 8 codes a thread 49, with two rows of each 45, with the codes loaded through the
// caches' reusable lines 45, with streaming stores 55.)
template <typename T, bool E4M3, int EPL>
__global__ void __launch_bounds__(256) kv_cache_read_kernel(const CacheParams p) {
  const int lane = threadIdx.x & 63;
  const int per_row = p.dim / EPL, per_token = p.kv_heads * per_row;
  const int64_t unit0 = (int64_t)blockIdx.x * 256;
  const int64_t token0 = unit0 / per_token;
  // the last sequence that starts at or before the workgroup's first token, -1 if none does; starts that
  // fall can name one that begins later, so the row's own place in it is looked at below
  int b = -1;
  for (int i = 0; i < p.batch; i += 64) {
    const bool below = i + lane < p.batch && p.starts[min(i + lane, p.batch - 1)] <= token0;
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(below));
    b += n;
    if (n < 64) break;
  }
  const int rest = (int)(unit0 - token0 * per_token) + (int)threadIdx.x;
  const int ahead = rest / per_token, within = rest - ahead * per_token;
  const int64_t token = token0 + ahead;
  if (token >= p.tokens) return;
  const int head = within / per_row, e = (within - head * per_row) * EPL;
  while (b + 1 < p.batch && p.starts[b + 1] <= token) ++b;
  u32x4 k[EPL / 8], v[EPL / 8];
#pragma unroll
  for (int h = 0; h < EPL / 8; ++h) k[h] = v[h] = u32x4{0, 0, 0, 0};
  if (b >= 0 && token < p.starts[b + 1]) {
    const int64_t key = token - p.starts[b];
    int place, page = -1;
    if (key >= 0 && key < (int64_t)p.kv.table_pages * p.kv.page_size)
      page = page_of(p.kv, p.kv.table + b * p.kv.table_row, (int)key, place);
    if (page >= 0) {
      float ks = 1.f, vs = 1.f;
      if constexpr (E4M3) {
        ks = p.kv.k_scale[page * p.kv.ks_page + place * p.kv.ks_token + head * p.kv.ks_head];
        vs = p.kv.v_scale[page * p.kv.vs_page + place * p.kv.vs_token + head * p.kv.vs_head];
      }
      read_row<T, E4M3, EPL>(p.kv.k, page * p.kv.k_page + place * p.kv.k_token + head * p.kv.k_head + e, ks, k);
      read_row<T, E4M3, EPL>(p.kv.v, page * p.kv.v_page + place * p.kv.v_token + head * p.kv.v_head + e, vs, v);
    }
  }
  const int64_t to = (token * p.kv_heads + head) * p.dim + e;
#pragma unroll
  for (int h = 0; h < EPL / 8; ++h) {
    *(u32x4*)((T*)p.k_out + to + 8 * h) = k[h];
    *(u32x4*)((T*)p.v_out + to + 8 * h) = v[h];
  }
}

template <typename T, bool E4M3>
static hipError_t launch_write(const CacheParams& p, hipStream_t s) {
  const int lanes = p.dim <= 64 ? 8 : p.dim <= 128 ? 16 : 32;
  const dim3 grid((unsigned)((p.tokens * p.kv_heads * lanes + 255) / 256)), block(256);
  if (lanes == 8) return launch_kernel(kv_cache_write_kernel<T, E4M3, 8>, grid, block, 0, s, p);
  if (lanes == 16) return launch_kernel(kv_cache_write_kernel<T, E4M3, 16>, grid, block, 0, s, p);
  return launch_kernel(kv_cache_write_kernel<T, E4M3, 32>, grid, block, 0, s, p);
}
template <typename T, bool E4M3>
static hipError_t launch_read(const CacheParams& p, hipStream_t s) {
  // 16 codes, or 8 elements, are 16 bytes; heads that are no multiple of 16 read 8 codes
  const int epl = E4M3 && p.dim % 16 == 0 ? 16 : 8;
  const dim3 grid((unsigned)((p.tokens * p.kv_heads * (p.dim / epl) + 255) / 256)), block(256);
  if constexpr (E4M3)
    if (epl == 16) return launch_kernel(kv_cache_read_kernel<T, true, 16>, grid, block, 0, s, p);
  return launch_kernel(kv_cache_read_kernel<T, E4M3, 8>, grid, block, 0, s, p);
}

hipError_t launch_kv_cache_write(int dtype, bool e4m3, const CacheParams& p, hipStream_t s) {
  if (dtype == kF16) return e4m3 ? launch_write<_Float16, true>(p, s) : launch_write<_Float16, false>(p, s);
  return e4m3 ? launch_write<__bf16, true>(p, s) : launch_write<__bf16, false>(p, s);
}
hipError_t launch_kv_cache_read(int dtype, bool e4m3, const CacheParams& p, hipStream_t s) {
  if (dtype == kF16) return e4m3 ? launch_read<_Float16, true>(p, s) : launch_read<_Float16, false>(p, s);
  return e4m3 ? launch_read<__bf16, true>(p, s) : launch_read<__bf16, false>(p, s);
}

}  // namespace cmpext3
