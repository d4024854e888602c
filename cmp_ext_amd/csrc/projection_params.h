// Kernel arguments and launchers of the feed-forward operators, shared by the host planner
// and the device code.  Row pitches are in elements.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

namespace cmpext3 {

// Element types as in the C ABI (dtype codes of GemmParams, and 8-bit codes).
constexpr int kI8 = 4;

// What a kernel computes from its one or two products.
enum ProjMode : int {
  kProjPlain = 0,  // sum_k a b, scaled (8-bit codes), plus the bias
  kProjGated = 1,  // act(sum_k a b0) * (sum_k a b1)
  kProjSum = 2,    // sum_k a0 b0 + sum_k a1 b1
};

struct ProjParams {
  const void* a[2];  // kProjSum: both; otherwise a[0]
  const void* b[2];  // kProjPlain: b[0]
  int64_t lda, ldb[2];
  const float* a_scale;     // 8-bit codes: of a row of a,
  const float* b_scale[2];  // of a row of b
  const void* bias;         // kProjPlain: [N] of the output's type, or nullptr
  void* out;
  int64_t ldo;
  int out_dtype;  // kF16, kBF16, kF32
  float* pre[2];  // kProjGated: both products, or nullptr
  int64_t ld_pre;
  int act;
  int M, N, K;
  int64_t batch_a, batch_out;  // grid.z: what a further product adds to a (elements) and out
};

// Any pitch and alignment; a is [M, K] or, a_km, [K, M]; b is [N, K] or, b_kn, [K, N].
hipError_t launch_projection_any(int dtype, ProjMode mode, bool a_km, bool b_kn, const ProjParams& p, hipStream_t s);

struct QuantParams {
  const void* x;
  int64_t ldx;
  int8_t* codes;
  int64_t ldc;
  float* scale;
  int64_t rows;
  int cols;
};
hipError_t launch_quantize_int8(int dtype, const QuantParams& p, hipStream_t s);

// dgate = grad * up * act'(gate), dup = grad * act(gate): [M, N] each, rows of ld_d elements of
// which those past N are set to zero.
struct GatedGradParams {
  const void* grad;
  const float* gate;
  const float* up;
  void* dgate;
  void* dup;
  int64_t ld_grad, ld_pre, ld_d;
  int act, M, N;
};
hipError_t launch_gated_grad(int dtype, const GatedGradParams& p, hipStream_t s);

}  // namespace cmpext3
