// The gradients of a gated block's two products, from that of their result:
//   dgate = grad * up * act'(gate),   dup = grad * act(gate),
// in fp32, rounded to 16 bits as the operands of the products that follow.  Both products come in
// fp32: held in 16 bits they would make the gradients' error 1.8 times that of rounding the result
// (as it is 1.4 times, from the rounding of dgate and dup alone), for 4 % of a training step's time.
//
// bf16 has fp32's range.  f16 ends at 65504 and at 2^-24, and a product of two or three of its values does not, while the
// sums that follow may well be inside.  So f16 holds dgate and dup times powers of two, which the products' last step
// takes out again: for dx, a sum over a row, each row's largest value is put between 2^14 and 2^15; for the weights, sums over
// a column, each column's.  (One unit for all would take the digits of every token beside one of large gradients.)  The two
// copies, and the pass that looks for the largest, are what f16 pays: a training step of 4096 x 4096, two of 14336, 2.50 ms for
// bf16's 2.20, of which the pass takes 126 us, the units 5 and the second copies 45; 500 x 1024, two of 2816, captured, 66 us for 55.
//
// Bound by HBM: bf16 [4096, 14336] 822 MB in 137 us, 6.0 TB/s; what is read once is read past the reusable lines, which
// the products that follow want for dgate and dup (174 us without).
#include "projection_common.h"

namespace cmpext3 {
namespace {

// Eight columns of a row, from n, zeros past N.  Rows of grad, gate and up may start at any element.
struct Eight {
  u32x4 d;
  f32x4 g[2], u[2];
  template <bool ONCE>
  __device__ __forceinline__ void load(const GatedGradParams& p, int64_t m, int64_t n) {
    typedef u32x4 u32x4_e __attribute__((aligned(2)));
    typedef f32x4 f32x4_e __attribute__((aligned(4)));
    const uint16_t* grad = (const uint16_t*)p.grad + m * p.ld_grad + n;
    const float* gate = p.gate + m * p.ld_pre + n;
    const float* up = p.up + m * p.ld_pre + n;
    auto get = [](auto* from) {
      if constexpr (ONCE) return __builtin_nontemporal_load(from);
      else return *from;
    };
    d = u32x4{0, 0, 0, 0};
    if (n + 8 <= p.N) {
      d = get((const u32x4_e*)grad);
#pragma unroll
      for (int h = 0; h < 2; ++h) g[h] = get((const f32x4_e*)(gate + 4 * h)), u[h] = get((const f32x4_e*)(up + 4 * h));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = n + i < p.N;
        if (in) d[i >> 1] |= (uint32_t)grad[i] << (16 * (i & 1));
        g[i >> 2][i & 3] = in ? gate[i] : 0.f;
        u[i >> 2][i & 3] = in ? up[i] : 0.f;
      }
    }
  }
  // dgate's in a, dup's in b
  template <typename T, int ACT>
  __device__ __forceinline__ void gradients(float* a, float* b) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float x = from_bits<T>((uint16_t)(d[k >> 1] >> (16 * (k & 1))));
      float value, slope;
      act_both<ACT>(g[k >> 2][k & 3], value, slope);
      a[k] = x * u[k >> 2][k & 3] * slope;
      b[k] = x * value;
    }
  }
};

// A thread takes eight columns of a row; rows of the results are whole 16 bytes.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) gated_grad_kernel(const GatedGradParams p) {
  constexpr bool UNITS = std::is_same<T, _Float16>::value;
  const int blocks = (int)((p.ld_d + 2047) / 2048);  // of a row
  const int64_t m = blockIdx.x / blocks;
  const int64_t n = ((int64_t)(blockIdx.x % blocks) * 256 + threadIdx.x) * 8;
  if (n >= p.ld_d) return;
  Eight in;
  in.load<true>(p, m, n);
  float v[2][8];
  in.gradients<T, ACT>(v[0], v[1]);
  auto store = [&](void* to, const float* x) {
    u32x4 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
    *(u32x4*)((uint16_t*)to + m * p.ld_d + n) = h;
  };
  const float row = UNITS ? p.units.row[m] : 1.f;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float x[8];
    if (!UNITS || p.d[q] != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = UNITS ? v[q][i] * row : v[q][i];
      store(p.d[q], x);
    }
    if (UNITS && p.d_col[q] != nullptr) {
      const f32x4* unit = (const f32x4*)(p.units.col + q * p.ld_d + n);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = v[q][i] * unit[i >> 2][i & 3];
      store(p.d_col[q], x);
    }
  }
}

// ---- f16: the units ----

// A finite value's bits without the sign, ordered as the values are; 0 for others, whose rows and columns are not
// finite whatever the unit.
__device__ __forceinline__ uint32_t size_of(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return a > b ? a : b; }

// A workgroup takes 512 columns of a block of rows, a wave two rows of every eight: both are on their way at once.
// ONCE: read past the reusable lines, where the next kernel would find none of it (see launch_act).
template <int ACT, bool ONCE>
__global__ void __launch_bounds__(256) gated_grad_most_kernel(const GatedGradParams p) {
  __shared__ uint32_t all[4][16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int cb = (int)(blockIdx.x % p.units.col_blocks), rb = (int)(blockIdx.x / p.units.col_blocks);
  const int64_t n = (int64_t)cb * kGradBlockCols + 8 * lane;
  const int64_t first = (int64_t)rb * p.units.rows_of_block;
  const int64_t end = first + p.units.rows_of_block < p.M ? first + p.units.rows_of_block : p.M;
  uint32_t cols[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) cols[i] = 0;
  for (int64_t m = first + 2 * wave; m < end; m += 8) {
    const bool two = m + 1 < end;
    Eight in[2];
    in[0].load<ONCE>(p, m, n);
    in[1].load<ONCE>(p, two ? m + 1 : m, n);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float v[2][8];
      in[r].gradients<_Float16, ACT>(v[0], v[1]);
      uint32_t of_row = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t b = size_of(v[i >> 3][i & 7]);
        cols[i] = most(cols[i], b);
        of_row = most(of_row, b);
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) of_row = most(of_row, (uint32_t)__shfl_xor((int)of_row, d));
      if (lane == 0) p.units.row_most[(int64_t)cb * p.M + (r == 0 || !two ? m : m + 1)] = of_row;
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) all[wave][i][lane] = cols[i];
  __syncthreads();
  // thread t: columns of product t / 128, four from 4 (t % 128) of the block
  const int q = threadIdx.x >> 7, c = 4 * (threadIdx.x & 127);
  const int64_t at = (int64_t)cb * kGradBlockCols + c;
  if (at >= p.ld_d) return;
  u32x4 of_col;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    of_col[i] = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) of_col[i] = most(of_col[i], all[w][8 * q + (c & 4) + i][c >> 3]);
  }
  *(u32x4*)(p.units.col_most + ((int64_t)rb * 2 + q) * p.ld_d + at) = of_col;
}

// The power of two that puts a value of these bits between 2^14 and 2^15, and its inverse; nothing but zeros: 1.  2^64 at most:
// what then still loses digits is below 2^-78, and 2^21 such terms times 2^16 do not reach f16's last digit.
__device__ __forceinline__ void unit_of(uint32_t bits, float* unit, float* inverse) {
  const int up = bits == 0 ? 0 : min(14 + 127 - (int)(bits >> 23), 64);  // -113 at least
  *unit = __uint_as_float((uint32_t)(127 + up) << 23);
  *inverse = __uint_as_float((uint32_t)(127 - up) << 23);
}

// A workgroup takes 32 rows or columns, eight threads each a share of the blocks: there may be hundreds, and few workgroups.
constexpr int kUnitsOfBlock = 32;
__global__ void __launch_bounds__(256) gated_grad_units_kernel(const GatedGradParams p) {
  __shared__ uint32_t all[8][kUnitsOfBlock];
  const int part = threadIdx.x / kUnitsOfBlock, c = threadIdx.x % kUnitsOfBlock;
  const int64_t t = (int64_t)blockIdx.x * kUnitsOfBlock + c;
  const bool row = t < p.M, col = !row && t < p.M + 2 * p.ld_d;
  const uint32_t* from = row ? p.units.row_most + t : p.units.col_most + (t - p.M);
  const int64_t pitch = row ? p.M : 2 * p.ld_d;
  const int count = row ? p.units.col_blocks : col ? p.units.row_blocks : 0;
  uint32_t bits = 0;
#pragma unroll 8
  for (int i = part; i < count; i += 8) bits = most(bits, from[i * pitch]);
  all[part][c] = bits;
  __syncthreads();
  if (part > 0) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) bits = most(bits, all[i][c]);
  float unit, inverse;
  unit_of(bits, &unit, &inverse);
  if (row) {
    p.units.row[t] = unit;
    p.units.row_inverse[t] = inverse;
  } else if (col) {
    const int64_t j = t - p.M;
    const int q = j >= p.ld_d;
    const int64_t n = j - q * p.ld_d;
    p.units.col[j] = unit;
    if (n < p.N) p.units.col_inverse[q * (int64_t)p.N + n] = inverse;
  }
}

template <typename T, int ACT>
hipError_t launch_act(const GatedGradParams& p, hipStream_t s) {
  const dim3 block(256);
  if constexpr (std::is_same<T, _Float16>::value) {
    // What the 256 MB of the Infinity Cache hold is read again from there: a training step of [4096, 14336] 2526 us without
    // ONCE and 2496 with it, but [4096, 4096] 730 and 747, [2048, 2816] 142 and 150.
    const dim3 grid((unsigned)(p.units.col_blocks * p.units.row_blocks));
    const bool once = (int64_t)p.M * p.N * 10 > 256ll << 20;
    hipError_t e = once ? launch_kernel((gated_grad_most_kernel<ACT, true>), grid, block, 0, s, p)
                        : launch_kernel((gated_grad_most_kernel<ACT, false>), grid, block, 0, s, p);
    if (e == hipSuccess) e = launch_kernel(gated_grad_units_kernel, dim3((unsigned)((p.M + 2 * p.ld_d + kUnitsOfBlock - 1) / kUnitsOfBlock)), block, 0, s, p);
    if (e != hipSuccess) return e;
  }
  return launch_kernel((gated_grad_kernel<T, ACT>), dim3((unsigned)(p.M * ((p.ld_d + 2047) / 2048))), block, 0, s, p);
}

template <typename T>
hipError_t launch(const GatedGradParams& p, hipStream_t s) {
  switch (p.act) {
    case CMPEXT3_ACT_SILU: return launch_act<T, CMPEXT3_ACT_SILU>(p, s);
    case CMPEXT3_ACT_GELU: return launch_act<T, CMPEXT3_ACT_GELU>(p, s);
    case CMPEXT3_ACT_GELU_TANH: return launch_act<T, CMPEXT3_ACT_GELU_TANH>(p, s);
    default: return launch_act<T, CMPEXT3_ACT_RELU>(p, s);
  }
}

}  // namespace

hipError_t launch_gated_grad(int dtype, const GatedGradParams& p, hipStream_t s) {
  return dtype == kF16 ? launch<_Float16>(p, s) : launch<__bf16>(p, s);
}

}  // namespace cmpext3
