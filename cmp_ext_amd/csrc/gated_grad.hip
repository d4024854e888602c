// The gradients of a gated block's two products, from that of their result:
//   dgate = grad * up * act'(gate),   dup = grad * act(gate),
// in fp32, rounded to 16 bits as the operands of the products that follow.  Both products come in
// fp32: held in 16 bits they would make the gradients' error 1.8 times that of rounding the result
// (as it is 1.4 times, from the rounding of dgate and dup alone), for 4 % of a training step's time.
//
// Bound by HBM: [4096, 14336] 822 MB in 137 us, 6.0 TB/s; what is read once is read past the reusable lines, which
// the products that follow want for dgate and dup (174 us without).
#include "projection_common.h"

namespace cmpext3 {
namespace {

// A thread takes eight columns of a row.  Rows of grad, gate and up may start at any element; those of dgate and
// dup are whole 16 bytes.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) gated_grad_kernel(const GatedGradParams p) {
  typedef u32x4 u32x4_e __attribute__((aligned(2)));
  typedef f32x4 f32x4_e __attribute__((aligned(4)));
  const int blocks = (int)((p.ld_d + 2047) / 2048);  // of a row
  const int64_t m = blockIdx.x / blocks;
  const int64_t n = ((int64_t)(blockIdx.x % blocks) * 256 + threadIdx.x) * 8;
  if (n >= p.ld_d) return;
  const uint16_t* grad = (const uint16_t*)p.grad + m * p.ld_grad + n;
  const float* gate = p.gate + m * p.ld_pre + n;
  const float* up = p.up + m * p.ld_pre + n;
  u32x4 d = {0, 0, 0, 0};
  f32x4 g[2], u[2];
  if (n + 8 <= p.N) {
    d = __builtin_nontemporal_load((const u32x4_e*)grad);
#pragma unroll
    for (int h = 0; h < 2; ++h) g[h] = __builtin_nontemporal_load((const f32x4_e*)(gate + 4 * h)), u[h] = __builtin_nontemporal_load((const f32x4_e*)(up + 4 * h));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = n + i < p.N;
      if (in) d[i >> 1] |= (uint32_t)grad[i] << (16 * (i & 1));
      g[i >> 2][i & 3] = in ? gate[i] : 0.f;
      u[i >> 2][i & 3] = in ? up[i] : 0.f;
    }
  }
  u32x4 dg, du;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a[2], b[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = 2 * i + e;
      const float x = from_bits<T>((uint16_t)(d[i] >> (16 * e)));
      float value, slope;
      act_both<ACT>(g[k >> 2][k & 3], value, slope);
      a[e] = x * u[k >> 2][k & 3] * slope;
      b[e] = x * value;
    }
    dg[i] = pack2<T>(a[0], a[1]);
    du[i] = pack2<T>(b[0], b[1]);
  }
  *(u32x4*)((uint16_t*)p.dgate + m * p.ld_d + n) = dg;
  *(u32x4*)((uint16_t*)p.dup + m * p.ld_d + n) = du;
}

template <typename T>
hipError_t launch(const GatedGradParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.M * ((p.ld_d + 2047) / 2048))), block(256);
  switch (p.act) {
    case CMPEXT3_ACT_SILU: return launch_kernel((gated_grad_kernel<T, CMPEXT3_ACT_SILU>), grid, block, 0, s, p);
    case CMPEXT3_ACT_GELU: return launch_kernel((gated_grad_kernel<T, CMPEXT3_ACT_GELU>), grid, block, 0, s, p);
    case CMPEXT3_ACT_GELU_TANH: return launch_kernel((gated_grad_kernel<T, CMPEXT3_ACT_GELU_TANH>), grid, block, 0, s, p);
    default: return launch_kernel((gated_grad_kernel<T, CMPEXT3_ACT_RELU>), grid, block, 0, s, p);
  }
}

}  // namespace

hipError_t launch_gated_grad(int dtype, const GatedGradParams& p, hipStream_t s) {
  return dtype == kF16 ? launch<_Float16>(p, s) : launch<__bf16>(p, s);
}

}  // namespace cmpext3
