// C ABI of the feed-forward operators (declared in include/cmpext3_projection.h): checks every
// argument, picks the kernels and launches them on the caller's stream.
#include <hip/hip_runtime_api.h>
#include <limits.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

#include "../../include/cmpext3_projection.h"
#include "gemm_params.h"
#include "projection_params.h"

using namespace cmpext3;

namespace {

constexpr int64_t kMostThreads = UINT32_MAX;  // of a grid, in one direction
constexpr int kMostGridY = 65535;
// Pitches that a tile's rows can be addressed with in 32-bit byte offsets.
constexpr int64_t kMaxPitch = INT_MAX / (256 * 4);

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }
bool is16(int dtype) { return dtype == CMPEXT3_F16 || dtype == CMPEXT3_BF16; }
size_t elem_size(int dtype) { return dtype == CMPEXT3_F32 ? 4 : dtype == CMPEXT3_I8 ? 1 : 2; }

// A matrix of `rows` rows of `cols` elements with the given pitch: its address (whole elements), pitch and size.
int check_matrix(const void* p, int64_t rows, int64_t cols, int64_t pitch, int dtype) {
  if (rows == 0 || cols == 0) return CMPEXT3_OK;
  if (p == nullptr || !aligned(p, elem_size(dtype)) || pitch < cols) return CMPEXT3_ERR_INVALID_ARG;
  return pitch > kMaxPitch ? CMPEXT3_ERR_TOO_LARGE : CMPEXT3_OK;
}

int first_of(std::initializer_list<int> checks) {
  for (int st : checks)
    if (st != CMPEXT3_OK) return st;
  return CMPEXT3_OK;
}

// Sizes that every grid and every 32-bit count in the kernels has room for, padding included.
int check_sizes(int M, int N, int K) {
  if (M < 0 || N < 0 || K < 0) return CMPEXT3_ERR_INVALID_ARG;
  const int most = INT_MAX - 512;
  if (M > most || N > most || K > most) return CMPEXT3_ERR_TOO_LARGE;
  return CMPEXT3_OK;
}
bool any_grid_fits(int64_t M, int64_t N) { return cdiv(M, 64) * 256 <= kMostThreads && cdiv(N, 64) <= kMostGridY; }

int check_workspace(int64_t need, const void* ws, int64_t bytes) {
  if (need < 0) return (int)need;
  if (need > 0 && (ws == nullptr || bytes < need || !aligned(ws, 16))) return CMPEXT3_ERR_WORKSPACE;
  return CMPEXT3_OK;
}

int check_projection(const cmpext3_projection_args* a) {
  if (a == nullptr) return CMPEXT3_ERR_INVALID_ARG;
  const bool i8 = a->dtype == CMPEXT3_I8, gated = a->w_up != nullptr;
  if (!i8 && !is16(a->dtype)) return CMPEXT3_ERR_UNSUPPORTED;
  if (!is16(a->out_dtype) && !(i8 && a->out_dtype == CMPEXT3_F32)) return CMPEXT3_ERR_UNSUPPORTED;
  if (!i8 && (a->out_dtype != a->dtype || !gated)) return CMPEXT3_ERR_UNSUPPORTED;
  if (gated && (a->activation < CMPEXT3_ACT_SILU || a->activation > CMPEXT3_ACT_RELU)) return CMPEXT3_ERR_UNSUPPORTED;
  if (gated && a->bias != nullptr) return CMPEXT3_ERR_UNSUPPORTED;
  if ((a->gate_out != nullptr) != (a->up_out != nullptr)) return CMPEXT3_ERR_INVALID_ARG;
  if (a->gate_out != nullptr && (i8 || !gated)) return CMPEXT3_ERR_UNSUPPORTED;
  int st = check_sizes(a->M, a->N, a->K);
  if (st != CMPEXT3_OK) return st;
  if (i8 && a->K > CMPEXT3_I8_MAX_K) return CMPEXT3_ERR_TOO_LARGE;
  if (a->M == 0 || a->N == 0) return CMPEXT3_OK;
  st = first_of({check_matrix(a->x, a->M, a->K, a->x_row, a->dtype), check_matrix(a->w_gate, a->N, a->K, a->gate_row, a->dtype),
                 gated ? check_matrix(a->w_up, a->N, a->K, a->up_row, a->dtype) : CMPEXT3_OK,
                 check_matrix(a->out, a->M, a->N, a->out_row, a->out_dtype)});
  if (st != CMPEXT3_OK) return st;
  if (a->gate_out != nullptr) {
    st = first_of({check_matrix(a->gate_out, a->M, a->N, a->pre_row, CMPEXT3_F32), check_matrix(a->up_out, a->M, a->N, a->pre_row, CMPEXT3_F32)});
    if (st != CMPEXT3_OK) return st;
  }
  if (i8) {
    if (a->x_scale == nullptr || !aligned(a->x_scale, 4)) return CMPEXT3_ERR_INVALID_ARG;
    if (a->gate_scale == nullptr || !aligned(a->gate_scale, 4)) return CMPEXT3_ERR_INVALID_ARG;
    if (gated && (a->up_scale == nullptr || !aligned(a->up_scale, 4))) return CMPEXT3_ERR_INVALID_ARG;
  }
  if (a->bias != nullptr && !aligned(a->bias, elem_size(a->out_dtype))) return CMPEXT3_ERR_INVALID_ARG;
  if (!any_grid_fits(a->M, a->N)) return CMPEXT3_ERR_TOO_LARGE;
  return CMPEXT3_OK;
}

ProjParams params_of(const cmpext3_projection_args* a) {
  ProjParams p{};
  p.a[0] = p.a[1] = a->x;
  p.b[0] = a->w_gate;
  p.b[1] = a->w_up;
  p.lda = a->x_row;
  p.ldb[0] = a->gate_row;
  p.ldb[1] = a->up_row;
  p.a_scale = a->x_scale;
  p.b_scale[0] = a->gate_scale;
  p.b_scale[1] = a->up_scale;
  p.bias = a->bias;
  p.out = a->out;
  p.ldo = a->out_row;
  p.out_dtype = a->out_dtype;
  p.pre[0] = a->gate_out;
  p.pre[1] = a->up_out;
  p.ld_pre = a->pre_row;
  p.act = a->activation;
  p.M = a->M, p.N = a->N, p.K = a->K;
  return p;
}

int check_gated_backward(const cmpext3_gated_backward_args* a) {
  if (a == nullptr) return CMPEXT3_ERR_INVALID_ARG;
  if (!is16(a->dtype)) return CMPEXT3_ERR_UNSUPPORTED;
  if (a->activation < CMPEXT3_ACT_SILU || a->activation > CMPEXT3_ACT_RELU) return CMPEXT3_ERR_UNSUPPORTED;
  int st = check_sizes(a->M, a->N, a->K);
  if (st != CMPEXT3_OK) return st;
  const int t = a->dtype;
  st = first_of({check_matrix(a->grad_out, a->M, a->N, a->grad_row, t), check_matrix(a->gate, a->M, a->N, a->pre_row, CMPEXT3_F32),
                 check_matrix(a->up, a->M, a->N, a->pre_row, CMPEXT3_F32)});
  if (st == CMPEXT3_OK && a->dx != nullptr)
    st = first_of({check_matrix(a->dx, a->M, a->K, a->dx_row, t), check_matrix(a->w_gate, a->N, a->K, a->gate_row, t),
                   check_matrix(a->w_up, a->N, a->K, a->up_row, t)});
  if (st == CMPEXT3_OK && (a->dw_gate != nullptr || a->dw_up != nullptr)) st = check_matrix(a->x, a->M, a->K, a->x_row, t);
  if (st == CMPEXT3_OK && a->dw_gate != nullptr) st = check_matrix(a->dw_gate, a->N, a->K, a->dgate_row, t);
  if (st == CMPEXT3_OK && a->dw_up != nullptr) st = check_matrix(a->dw_up, a->N, a->K, a->dup_row, t);
  if (st != CMPEXT3_OK) return st;
  if (!any_grid_fits(a->M, a->K) || !any_grid_fits(a->N, a->K)) return CMPEXT3_ERR_TOO_LARGE;
  if (a->M * (int64_t)256 > kMostThreads || cdiv(a->N, 256) >= kMostGridY) return CMPEXT3_ERR_TOO_LARGE;
  return CMPEXT3_OK;
}

// Elements of a row of the held gradients: whole 16 bytes.
int64_t grad_pitch(int N) { return cdiv(N, 8) * 8; }

}  // namespace

extern "C" int cmpext3_quantize_int8(const cmpext3_quantize_int8_args* a, void* stream) {
  if (a == nullptr) return CMPEXT3_ERR_INVALID_ARG;
  if (!is16(a->dtype) && a->dtype != CMPEXT3_F32) return CMPEXT3_ERR_UNSUPPORTED;
  if (a->rows < 0 || a->cols < 0) return CMPEXT3_ERR_INVALID_ARG;
  if (a->rows == 0) return CMPEXT3_OK;
  if (a->rows > kMostThreads / 256) return CMPEXT3_ERR_TOO_LARGE;
  if (a->scale == nullptr || !aligned(a->scale, 4)) return CMPEXT3_ERR_INVALID_ARG;
  if (a->cols > 0) {
    if (a->x == nullptr || a->codes == nullptr || !aligned(a->x, elem_size(a->dtype))) return CMPEXT3_ERR_INVALID_ARG;
    if (a->x_row < a->cols || a->codes_row < a->cols) return CMPEXT3_ERR_INVALID_ARG;
    if (a->x_row > INT64_MAX / 8 / a->rows || a->codes_row > INT64_MAX / 8 / a->rows) return CMPEXT3_ERR_TOO_LARGE;
  }
  QuantParams p{};
  p.x = a->x;
  p.ldx = a->x_row;
  p.codes = a->codes;
  p.ldc = a->codes_row;
  p.scale = a->scale;
  p.rows = a->rows;
  p.cols = a->cols;
  return (int)launch_quantize_int8(a->dtype, p, (hipStream_t)stream);
}

extern "C" int64_t cmpext3_projection_workspace_size(const cmpext3_projection_args* a) { return check_projection(a); }

extern "C" int cmpext3_projection(const cmpext3_projection_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t need = cmpext3_projection_workspace_size(a);
  const int st = check_workspace(need, workspace, workspace_bytes);
  if (st != CMPEXT3_OK) return st;
  if (a->M == 0 || a->N == 0) return CMPEXT3_OK;
  const ProjMode mode = a->w_up != nullptr ? kProjGated : kProjPlain;
  return (int)launch_projection_any(a->dtype, mode, false, false, params_of(a), (hipStream_t)stream);
}

extern "C" int cmpext3_projection_describe(const cmpext3_projection_args* a, char* buf, int buflen) {
  const int st = check_projection(a);
  if (st != CMPEXT3_OK) return st;
  if (buf != nullptr && buflen > 0) snprintf(buf, (size_t)buflen, "kernel=any64x64");
  return CMPEXT3_OK;
}

extern "C" int64_t cmpext3_gated_backward_workspace_size(const cmpext3_gated_backward_args* a) {
  const int st = check_gated_backward(a);
  if (st != CMPEXT3_OK) return st;
  return 2 * 2 * (int64_t)a->M * grad_pitch(a->N);
}

extern "C" int cmpext3_gated_backward(const cmpext3_gated_backward_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t need = cmpext3_gated_backward_workspace_size(a);
  const int st = check_workspace(need, workspace, workspace_bytes);
  if (st != CMPEXT3_OK) return st;
  const hipStream_t s = (hipStream_t)stream;
  const int64_t pitch = grad_pitch(a->N);
  uint16_t* d[2] = {(uint16_t*)workspace, (uint16_t*)workspace + (int64_t)a->M * pitch};
  hipError_t e = hipSuccess;
  if (a->M > 0 && a->N > 0) {
    GatedGradParams g{};
    g.grad = a->grad_out;
    g.gate = a->gate;
    g.up = a->up;
    g.dgate = d[0];
    g.dup = d[1];
    g.ld_grad = a->grad_row, g.ld_pre = a->pre_row, g.ld_d = pitch;
    g.act = a->activation;
    g.M = a->M, g.N = a->N;
    e = launch_gated_grad(a->dtype, g, s);
    if (e != hipSuccess) return (int)e;
  }
  ProjParams p{};
  p.out_dtype = a->dtype;
  p.lda = pitch;
  if (a->dx != nullptr && a->M > 0 && a->K > 0) {
    p.a[0] = d[0], p.a[1] = d[1];
    p.b[0] = a->w_gate, p.b[1] = a->w_up;
    p.ldb[0] = a->gate_row, p.ldb[1] = a->up_row;
    p.out = a->dx;
    p.ldo = a->dx_row;
    p.M = a->M, p.N = a->K, p.K = a->N;
    e = launch_projection_any(a->dtype, kProjSum, false, true, p, s);
    if (e != hipSuccess) return (int)e;
  }
  void* dw[2] = {a->dw_gate, a->dw_up};
  const int64_t dw_row[2] = {a->dgate_row, a->dup_row};
  for (int i = 0; i < 2; ++i) {
    if (dw[i] == nullptr || a->N == 0 || a->K == 0) continue;
    p.a[0] = d[i];
    p.b[0] = a->x;
    p.ldb[0] = a->x_row;
    p.out = dw[i];
    p.ldo = dw_row[i];
    p.M = a->N, p.N = a->K, p.K = a->M;
    e = launch_projection_any(a->dtype, kProjPlain, true, true, p, s);
    if (e != hipSuccess) return (int)e;
  }
  return CMPEXT3_OK;
}
