// The gradients of a gated block's two products, from that of their result:
//   dgate = grad * up * act'(gate),   dup = grad * act(gate),
// in fp32, rounded to 16 bits as the operands of the products that follow.  Both products come in
// fp32: held in 16 bits they would make the gradients' error 1.8 times that of rounding the result
// (as it is 1.4 times, from the rounding of dgate and dup alone), for 4 % of a training step's time.
#include "projection_common.h"

namespace cmpext3 {
namespace {

template <typename T, int ACT>
__global__ void __launch_bounds__(256) gated_grad_kernel(const GatedGradParams p) {
  const int64_t m = blockIdx.x;
  const int64_t n = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (n >= p.ld_d) return;
  uint16_t dg = 0, du = 0;
  if (n < p.N) {
    const float grad = from_bits<T>(((const uint16_t*)p.grad)[m * p.ld_grad + n]);
    const float up = p.up[m * p.ld_pre + n];
    float value, slope;
    act_both<ACT>(p.gate[m * p.ld_pre + n], value, slope);
    dg = to_bits<T>(grad * up * slope);
    du = to_bits<T>(grad * value);
  }
  ((uint16_t*)p.dgate)[m * p.ld_d + n] = dg;
  ((uint16_t*)p.dup)[m * p.ld_d + n] = du;
}

template <typename T>
hipError_t launch(const GatedGradParams& p, hipStream_t s) {
  const dim3 grid((unsigned)p.M, (unsigned)((p.ld_d + 255) / 256)), block(256);
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
