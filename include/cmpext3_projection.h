/*
 * cmpext3_projection.h -- C ABI of the feed-forward operators of the MI355X (gfx950)
 * library (libcmpext3_gemm.so): projections with weights in 8-bit integers, and the gated
 * first half of a feed-forward block with its backward pass.
 *
 * The conventions are those of cmpext3_gemm.h: device pointers owned by the caller, row
 * pitches in elements, no allocation, no synchronisation, work enqueued on `stream`,
 * CMPEXT3_OK or a CMPEXT3_ERR_* / hipError_t as the result, nothing launched when an
 * argument is rejected.  Matrices have rows of unit stride and a pitch of at least the row's
 * length; a structure that is cleared to zero before its fields are set stays valid when
 * fields are added behind the last one.
 */
#ifndef CMPEXT3_PROJECTION_H
#define CMPEXT3_PROJECTION_H

#include <stdint.h>

#include "cmpext3_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of codes: 8-bit signed integers. */
#define CMPEXT3_I8 4

/* Activations of a gated block. */
#define CMPEXT3_ACT_SILU 0      /* g / (1 + exp(-g))                                           */
#define CMPEXT3_ACT_GELU 1      /* g * P(Z <= g) for a normal Z: g / 2 * erfc(-g / sqrt(2))     */
#define CMPEXT3_ACT_GELU_TANH 2 /* g / 2 * (1 + tanh(sqrt(2 / pi) * (g + 0.044715 g^3)))        */
#define CMPEXT3_ACT_RELU 3      /* max(g, 0)                                                   */

/* Products over more terms than this could leave the 32-bit sums of 8-bit codes. */
#define CMPEXT3_I8_MAX_K 131071

/*
 * Rows of x [rows, cols] (F16, BF16 or F32) as 8-bit codes with one scale for each:
 *   a = max(max |x|, 2^-100),   code = round(127 x / a) (ties to even),   scale = a / 127
 * so that code * scale stands for x (F32: 127 x is rounded to fp32 first).  A row that holds NaN or an infinity gets
 * codes of 0 and a scale of NaN: whatever is computed from it is NaN.  cols up to 2^31 - 513.
 */
typedef struct cmpext3_quantize_int8_args {
  int32_t dtype;
  int32_t cols;
  int64_t rows;
  const void* x;
  int64_t x_row;
  int8_t* codes;
  int64_t codes_row;
  float* scale; /* [rows] */
} cmpext3_quantize_int8_args;
int cmpext3_quantize_int8(const cmpext3_quantize_int8_args* args, void* stream);

/*
 * One or two projections of x [M, K] by weights w [N, K]:
 *   plain (w_up NULL; dtype CMPEXT3_I8):  out = p(w) + bias
 *   gated (both weights):                 out = act(p(w_gate)) * p(w_up)
 * where p(w)[m, n] is the sum over k of x[m, k] * w[n, k]: F16 or BF16 with fp32 sums, or I8
 * with exact 32-bit integer sums times x_scale[m] and w_scale[n] (either may be large where the result is not).  x has x_dtype: that of the
 * weights, or, with I8 weights, F16, BF16 or F32: it is then taken as cmpext3_quantize_int8 would
 * give it (x_scale NULL).  out [M, N] has out_dtype (F16,
 * BF16, F32; that of x where it is not I8), rounded once.  In the plain form the weight is
 * w_gate, its scale gate_scale; bias [N] has out_dtype, or is NULL.  gate_out and up_out
 * (gated F16 / BF16 only; both or neither): p(w_gate) and p(w_up) as fp32, for the backward pass.
 * K = 0 gives sums of zero; K of I8 up to CMPEXT3_I8_MAX_K.
 */
typedef struct cmpext3_projection_args {
  int32_t dtype, x_dtype, out_dtype, activation; /* dtype: of the weights */
  int32_t M, N, K;
  const void* x;
  int64_t x_row;
  const float* x_scale; /* [M], x of I8 only */
  const void* w_gate;
  int64_t gate_row;
  const float* gate_scale; /* [N], I8 only */
  const void* w_up;
  int64_t up_row;
  const float* up_scale; /* [N], I8 only */
  const void* bias;
  void* out;
  int64_t out_row;
  float* gate_out;
  float* up_out;
  int64_t pre_row; /* of gate_out and up_out */
} cmpext3_projection_args;

/* Bytes of workspace (16-byte aligned) the call needs, often 0; or a CMPEXT3_ERR_*. */
int64_t cmpext3_projection_workspace_size(const cmpext3_projection_args* args);
int cmpext3_projection(const cmpext3_projection_args* args, void* workspace, int64_t workspace_bytes, void* stream);
/* Names the kernel, tile and split into buf. */
int cmpext3_projection_describe(const cmpext3_projection_args* args, char* buf, int buflen);

/*
 * The backward pass of a gated projection: from grad_out [M, N], the gradient of its output,
 * and gate, up [M, N], its two products as gate_out and up_out gave them (fp32),
 *   dgate = grad_out * up * act'(gate),   dup = grad_out * act(gate)    (fp32, rounded to dtype)
 *   dx      [M, K] = dgate w_gate + dup w_up         (one fp32 sum over both)
 *   dw_gate [N, K] = dgate^T x,   dw_up [N, K] = dup^T x
 * dtype F16 or BF16 for all others; any of dx, dw_gate, dw_up may be NULL and is then not computed.
 * M = 0 gives weight gradients of zero.  The derivative of relu at 0 is 0.
 * F16 holds dgate and dup times powers of two, of each row for dx and of each channel for dw_gate and dw_up, which the
 * products take out again: neither need lie in the range of F16 (those below 2^-29 of their row's or channel's largest
 * lose digits).  The workspace holds dgate and dup: 4 bytes a result, F16 8 where dx and both dw are asked for.
 */
typedef struct cmpext3_gated_backward_args {
  int32_t dtype, activation;
  int32_t M, N, K;
  const void* grad_out;
  int64_t grad_row;
  const float* gate;
  const float* up;
  int64_t pre_row; /* of gate and up */
  const void* x;   /* needed for dw_gate and dw_up */
  int64_t x_row;
  const void* w_gate; /* needed for dx */
  int64_t gate_row;
  const void* w_up;
  int64_t up_row;
  void* dx;
  int64_t dx_row;
  void* dw_gate;
  int64_t dgate_row;
  void* dw_up;
  int64_t dup_row;
} cmpext3_gated_backward_args;
int64_t cmpext3_gated_backward_workspace_size(const cmpext3_gated_backward_args* args);
int cmpext3_gated_backward(const cmpext3_gated_backward_args* args, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CMPEXT3_PROJECTION_H */
