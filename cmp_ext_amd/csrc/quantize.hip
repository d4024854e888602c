// Rows as 8-bit codes with a scale for each: a = max(max |x|, 2^-100), code = round(127 x / a), scale = a / 127.
//
// Bound by reading x and writing the codes.  A wave takes a row of up to 2048 elements, a workgroup one of up to
// 16384, and holds it in registers between the search for its largest value and the codes, so that it
// is read once; longer rows are read twice (the second time mostly from the caches).  Pieces of 8 elements are loaded
// and stored whole at any alignment, but for a row's last.  [4096, 14336] bf16: 29.5 us (of which x may still be in the
// Infinity Cache; 5.9 TB/s), [16, 8192] 4.3, [1, 4096] 2.4.
#include "quantize_common.h"

namespace cmpext3 {
namespace {

// LANES: of a row, 64, 256 or 1024; PER: pieces of 8 elements that a lane holds, 0: the row is read twice.
template <typename T, int LANES, int PER>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) quantize_int8_kernel(const QuantParams p) {
  const int64_t row = LANES < 256 ? (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES : blockIdx.x;
  const int t = threadIdx.x % LANES;
  if (LANES == 64 && row >= p.rows) return;  // whole waves
  const T* x = (const T*)p.x + row * p.ldx;
  const int pieces = (p.written + 7) / 8;
  Piece<T> held[PER > 0 ? PER : 1];
  uint32_t most = 0;
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = t + LANES * i;
      held[i].load(x + 8 * (int64_t)at, p.cols - 8 * at);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) most = most_of(held[i], most);
  } else {
    for (int at = t; at < pieces; at += LANES) {
      held[0].load(x + 8 * (int64_t)at, p.cols - 8 * at);
      most = most_of(held[0], most);
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const uint32_t b = __shfl_xor(most, d);
    most = most > b ? most : b;
  }
  if constexpr (LANES > 64) {
    __shared__ uint32_t waves[LANES / 64];
    if ((t & 63) == 0) waves[t >> 6] = most;
    __syncthreads();
    most = waves[0];
#pragma unroll
    for (int i = 1; i < LANES / 64; ++i) most = most > waves[i] ? most : waves[i];
  }
  const RowScale r(most);
  if (t == 0) p.scale[row] = r.scale;
  int8_t* codes = p.codes + row * p.ldc;
  typedef u32x2 Any __attribute__((aligned(1)));
  auto store = [&](const Piece<T>& h, int at) {
    const u32x2 c = eight_codes(h, r);
    const int left = p.written - 8 * at;  // zeros past cols
    int8_t* dst = codes + 8 * (int64_t)at;
    if (left >= 8) {
      *(Any*)dst = c;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) dst[i] = (int8_t)(c[i >> 2] >> (8 * (i & 3)));
    }
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (t + LANES * i < pieces) store(held[i], t + LANES * i);
  } else {
    for (int at = t; at < pieces; at += LANES) {
      held[0].load(x + 8 * (int64_t)at, p.cols - 8 * at);
      store(held[0], at);
    }
  }
}

template <typename T>
hipError_t launch(const QuantParams& p, hipStream_t s) {
  const dim3 block(256), rows1((unsigned)p.rows), rows4((unsigned)((p.rows + 3) / 4));
  const int pieces = (p.written + 7) / 8;
  // a wave a row where rows are short, but a workgroup where they are few: its loads are all on their way at once
  if (p.rows >= 1024 || pieces <= 64) {
    if (pieces <= 64) return launch_kernel((quantize_int8_kernel<T, 64, 1>), rows4, block, 0, s, p);
    if (pieces <= 128) return launch_kernel((quantize_int8_kernel<T, 64, 2>), rows4, block, 0, s, p);
    if (pieces <= 256) return launch_kernel((quantize_int8_kernel<T, 64, 4>), rows4, block, 0, s, p);
  }
  if (p.rows <= 256 && pieces > 512) {  // rows of few workgroups: every piece has a lane
    if (pieces <= 1024) return launch_kernel((quantize_int8_kernel<T, 1024, 1>), rows1, dim3(1024), 0, s, p);
    if (pieces <= 2048) return launch_kernel((quantize_int8_kernel<T, 1024, 2>), rows1, dim3(1024), 0, s, p);
  }
  if (pieces <= 256) return launch_kernel((quantize_int8_kernel<T, 256, 1>), rows1, block, 0, s, p);
  if (pieces <= 512) return launch_kernel((quantize_int8_kernel<T, 256, 2>), rows1, block, 0, s, p);
  if (pieces <= 1024) return launch_kernel((quantize_int8_kernel<T, 256, 4>), rows1, block, 0, s, p);
  if (pieces <= 2048) return launch_kernel((quantize_int8_kernel<T, 256, 8>), rows1, block, 0, s, p);
  return launch_kernel((quantize_int8_kernel<T, 256, 0>), rows1, block, 0, s, p);
}

}  // namespace

hipError_t launch_quantize_int8(int dtype, const QuantParams& p, hipStream_t s) {
  if (dtype == kF16) return launch<_Float16>(p, s);
  if (dtype == kBF16) return launch<__bf16>(p, s);
  return launch<float>(p, s);
}

}  // namespace cmpext3
