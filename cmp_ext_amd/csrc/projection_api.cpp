// C ABI of the feed-forward operators (declared in include/cmpext3_projection.h): checks every
// argument, picks the kernels and launches them on the caller's stream.
#include <hip/hip_runtime_api.h>
#include <limits.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

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
constexpr int kMostSize = INT_MAX - 512;
int check_sizes(int M, int N, int K) {
  if (M < 0 || N < 0 || K < 0) return CMPEXT3_ERR_INVALID_ARG;
  if (M > kMostSize || N > kMostSize || K > kMostSize) return CMPEXT3_ERR_TOO_LARGE;
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
  if (a->x_dtype != a->dtype && !(i8 && (is16(a->x_dtype) || a->x_dtype == CMPEXT3_F32))) return CMPEXT3_ERR_UNSUPPORTED;
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
  st = first_of({check_matrix(a->x, a->M, a->K, a->x_row, a->x_dtype), check_matrix(a->w_gate, a->N, a->K, a->gate_row, a->dtype),
                 gated ? check_matrix(a->w_up, a->N, a->K, a->up_row, a->dtype) : CMPEXT3_OK,
                 check_matrix(a->out, a->M, a->N, a->out_row, a->out_dtype)});
  if (st != CMPEXT3_OK) return st;
  if (a->gate_out != nullptr) {
    st = first_of({check_matrix(a->gate_out, a->M, a->N, a->pre_row, CMPEXT3_F32), check_matrix(a->up_out, a->M, a->N, a->pre_row, CMPEXT3_F32)});
    if (st != CMPEXT3_OK) return st;
  }
  if (i8) {
    if ((a->x_scale != nullptr) != (a->x_dtype == CMPEXT3_I8) || !aligned(a->x_scale, 4)) return CMPEXT3_ERR_INVALID_ARG;
    if (a->x_dtype != CMPEXT3_I8 && a->M > kMostThreads / 256) return CMPEXT3_ERR_TOO_LARGE;
    if (a->gate_scale == nullptr || !aligned(a->gate_scale, 4)) return CMPEXT3_ERR_INVALID_ARG;
    if (gated && (a->up_scale == nullptr || !aligned(a->up_scale, 4))) return CMPEXT3_ERR_INVALID_ARG;
  }
  if (a->bias != nullptr && !aligned(a->bias, elem_size(a->out_dtype))) return CMPEXT3_ERR_INVALID_ARG;
  if (!any_grid_fits(a->M, a->N)) return CMPEXT3_ERR_TOO_LARGE;
  return CMPEXT3_OK;
}

// A matrix with rows along k that the tiles read: as it is, or as a copy in the workspace whose rows are whole
// 16 bytes, zero past the matrix.
struct Operand {
  const void* p;
  int64_t ld;
  int rows, cols;
  int64_t copy_at;  // in the workspace, or -1
  int64_t copy_ld;
};

bool rows_of_16(const Operand& o, size_t esz) {
  return aligned(o.p, 16) && (o.rows <= 1 || o.ld * (int64_t)esz % 16 == 0) && o.cols * (int64_t)esz % 16 == 0;
}

// Takes `bytes` of the workspace, in whole 256 bytes.
int64_t take(int64_t* used, int64_t bytes) {
  const int64_t at = *used;
  *used += cdiv(bytes, 256) * 256;
  return at;
}

void plan_copy(Operand* o, size_t esz, int64_t* used) {
  o->copy_at = -1;
  if (rows_of_16(*o, esz)) return;
  o->copy_ld = cdiv(o->cols * (int64_t)esz, 16) * 16 / (int64_t)esz;
  o->copy_at = take(used, (int64_t)o->rows * o->copy_ld * (int64_t)esz);
}

// Makes the operands' copies; afterwards the operands are the copies.
hipError_t run_copies(std::initializer_list<Operand*> operands, size_t esz, char* ws, hipStream_t s) {
  PadParams p{};
  int count = 0;
  for (Operand* o : operands) {
    if (o->copy_at < 0) continue;
    p.m[count++] = PadParams::Matrix{o->p, ws + o->copy_at, o->ld * (int64_t)esz, o->copy_ld * (int64_t)esz, o->rows, (int)(o->cols * (int64_t)esz)};
    o->p = ws + o->copy_at;
    o->ld = o->copy_ld;
  }
  return launch_projection_pad(p, count, s);
}

// Tuning override: CMPEXT3_PROJECTION_CONFIG="kernel=<any64x64|rows|small64x64|tile128x128|tile256x128|tile256x256>[,splits=<s>
// [,groups=<g>]]" replaces the plan's choice wherever that kernel can run.  For sweeps and tests: read on every plan,
// ignored where malformed.
struct Override {
  char kernel[32];
  int splits, groups;
  bool is(const char* name) const { return strcmp(kernel, name) == 0; }
  bool tiles() const { return is("small64x64") || is("tile128x128") || is("tile256x128") || is("tile256x256"); }
};
Override read_override() {
  Override o{};
  const char* env = getenv("CMPEXT3_PROJECTION_CONFIG");
  if (env != nullptr && sscanf(env, "kernel=%31[^,],splits=%d,groups=%d", o.kernel, &o.splits, &o.groups) < 1) o.kernel[0] = 0;
  return o;
}

struct TilePlan {
  int bm, bn;  // 256 x 256, 256 x 128, 128 x 128, 64 x 64 (no copies of operands), or 0: the kernel for any size
  bool deep;
  int groups;  // of four waves that share a 64 x 64 tile's steps
  int splits, ksplit;
};

// Which tiles, and in how many splits of the steps of 128 bytes of k, for M x N results (of `products` products)
// in `batch` entries; copy_us: what the large tiles' copies of operands take (0: none); rows16:
// operands' rows have 16 bytes, which copies and 64 x 64 tiles need; along: both operands along k.  Modelled microseconds, fitted
// to timings of some 60 shapes with every tile and 1, 2, 4 and 8 splits (MI355X): a round of workgroups takes its steps
// and some start and end, but no less than reading the operands once; splits add their sums' way to memory and back
// and a launch.  64 x 64 tiles run three to a CU, and read operands of odd rows (every line twice) at 0.9 us
// a step for 0.65: x[1000, 2001], two of 4001 rows, 90 us, in copies 67; x[333, 2050] by 1001 rows of codes 11.4 and 26.6,
// x[100, 1024], two of 1024, 8.5 for 10.0.  Where they are alone on their CUs two groups of waves share a tile's steps (256 x
// 4096 x 4096 of codes 14.8 -> 12.5 us, 128 x 4096 x 4096 14.1 -> 11.7, dx[64, 1024] 17.4 -> 14.6; four groups: no faster; but
// 8 steps 8.9 -> 11.9, and 2 tiles on some CUs no longer fit at once).
TilePlan plan_tiles(int64_t M, int64_t N, int64_t steps, int products, int64_t batch, double copy_us, bool rows16, bool along) {
  const Override o = read_override();
  TilePlan best{0, 0, false, 1, 1, (int)steps};
  double least = 1e30;
  auto consider = [&](int bm, int bn, const char* name) {
    if (((bm == 64 || copy_us > 0) && !rows16) || (bm != bn && !along) || (o.tiles() && !o.is(name))) return;
    const int64_t tiles = cdiv(M, bm) * cdiv(N, bn / products) * batch;
    for (int64_t s = 1; s <= 16 && (s == 1 || (s * 4 <= steps && bm < 256)); ++s) {
      const int64_t each = cdiv(steps, s);
      if (s > 1 && (s - 1) * each >= steps) continue;  // an empty split
      if (o.tiles() && o.splits > 0 && s != o.splits) continue;
      const int64_t wgs = tiles * s;
      if (wgs > kMostThreads / 512) break;
      bool deep = false;
      int groups = 1;
      double t = 0;
      if (bm == 256) {
        t += (double)cdiv(wgs, 256) * (bn == 256 ? each * 1.5 + 6.0 : wgs <= 224 ? each * 0.66 + 4.0 : each * 0.88 + 5.0);
      } else if (bm == 128) {
        deep = wgs <= 256 && each >= 8;
        const int64_t full = wgs / 512, rest = wgs % 512;
        t += (double)full * (each * 0.94 + 5.0);
        if (rest > 256) t += each * 0.94 + 5.0;
        else if (rest > 0) t += each * (!deep ? 0.70 : rest > 128 ? 0.40 : 0.33) + 5.0;
      } else {
        groups = wgs <= 256 && each >= 16 ? 2 : 1;
        if (o.groups > 0) groups = o.groups == 2 ? 2 : 1;
        const int64_t full = wgs / 768, rest = wgs % 768;
        const double busy = copy_us > 0 ? 0.9 : 0.65;
        t += (double)full * (each * busy + 4.0);
        if (rest > 0) t += each * (rest > 512 ? busy : rest > 256 ? 0.47 : groups == 2 ? 0.21 : 0.28) + 4.0;
      }
      t = std::max(t, (double)batch * (M + N * products) * steps * 128 / (bm == bn ? 4.5e6 : 3.7e6));
      if (bm > 64) t += copy_us;
      if (s > 1) t += 4.0 + (double)s * batch * M * N * products * 8.0 / 5e6;
      if (t < least) {
        least = t;
        best = TilePlan{bm, bn, deep, groups, (int)s, (int)each};
      }
    }
  };
  consider(256, 256, "tile256x256");
  consider(256, 128, "tile256x128");
  consider(128, 128, "tile128x128");
  consider(64, 64, "small64x64");
  return best;
}

int64_t partial_pitch(int64_t N) { return cdiv(N, 4) * 4; }
int64_t partial_bytes(const TilePlan& t, int64_t M, int64_t N, int products, int64_t batch) {
  return t.splits > 1 ? (int64_t)t.splits * batch * products * M * partial_pitch(N) * 4 : 0;
}

// Microseconds of the zero-padded copies of operands, in one launch, 0 where none is needed.
double copy_us(std::initializer_list<const Operand*> operands, size_t esz) {
  double us = 0;
  for (const Operand* o : operands)
    if (!rows_of_16(*o, esz)) us += (double)o->rows * o->cols * (int)esz * 2.0 / 4e6;
  return us > 0 ? us + 4.0 : 0.0;
}

// Sets the tiles' grid in p and launches them, and the join of their splits.
hipError_t run_tiles(int dtype, ProjMode mode, ProjTileLaunch* large, const TilePlan& t, ProjParams& p, void* partials, hipStream_t s) {
  const int products = mode == kProjGated ? 2 : 1;
  p.tiles_m = (int)cdiv(p.M, t.bm);
  p.tiles_n = (int)cdiv(p.N, t.bn / products);
  p.group_m = 4;
  p.splits = t.splits;
  p.ksplit = t.ksplit;
  p.partials = partials;
  p.ld_part = partial_pitch(p.N);
  ProjSmallLaunch* small = dtype == CMPEXT3_F16    ? launch_projection_small_f16
                           : dtype == CMPEXT3_BF16 ? launch_projection_small_bf16
                                                   : launch_projection_small_int8;
  const hipError_t e = t.bm == 64 ? small(mode, p, t.groups, s) : large(p, t.bm, t.bn, t.deep, s);
  return e != hipSuccess || t.splits == 1 ? e : launch_projection_join(dtype, mode, p, s);
}

enum ProjKernel { kAny, kRows, kTile };

struct ProjPlan {
  ProjKernel kernel;
  bool make;         // x's codes are made in the workspace first, in rows of whole 16 bytes with zeros behind x's,
  bool make_inside;  // or by the kernel
  int64_t codes_at, scale_at;
  Operand x, w[2];
  TilePlan tile;
  int64_t partials_at, ws_bytes;
};

int plan_projection(const cmpext3_projection_args* a, ProjPlan* q) {
  const int st = check_projection(a);
  if (st != CMPEXT3_OK) return st;
  *q = ProjPlan{};
  if (a->M == 0 || a->N == 0) return CMPEXT3_OK;
  const size_t esz = elem_size(a->dtype);
  const int products = a->w_up != nullptr ? 2 : 1;
  q->x = Operand{a->x, a->x_row, a->M, a->K, -1, 0};
  q->w[0] = Operand{a->w_gate, a->gate_row, a->N, a->K, -1, 0};
  q->w[1] = Operand{a->w_up, a->up_row, a->N, a->K, -1, 0};
  q->make = a->x_dtype != a->dtype;
  if (q->make) {
    const int pitch = (int)(cdiv(a->K, 16) * 16);
    const bool few = is16(a->x_dtype) && a->M <= kRowsCodesRows && (int64_t)a->M * a->K <= kRowsCodesMost && a->K % kRowsCodesUnit == 0 && a->K > 0 &&
                     rows_of_16(q->x, elem_size(a->x_dtype));
    q->make_inside = few && rows_of_16(q->w[0], 1) && (products == 1 || rows_of_16(q->w[1], 1)) && read_override().kernel[0] == 0;
    if (q->make_inside) {
      q->kernel = kRows;
      return CMPEXT3_OK;
    }
    q->codes_at = take(&q->ws_bytes, (int64_t)a->M * pitch);
    q->scale_at = take(&q->ws_bytes, (int64_t)a->M * 4);
    q->x = Operand{nullptr, pitch, a->M, pitch, -1, 0};  // an address of 16 bytes: the workspace's
  }
  const Override o = read_override();
  const bool whole = rows_of_16(q->x, esz) && rows_of_16(q->w[0], esz) && (products == 1 || rows_of_16(q->w[1], esz));
  q->kernel = kAny;
  if ((int64_t)a->K * (int64_t)esz < 16 || o.is("any64x64")) return CMPEXT3_OK;
  // Few rows: bound by reading the weights, once.  Above 32 rows the 64 x 64 tiles are as fast where they fill the CUs
  // (codes, 64 x 4096 x 14336: 16.1 us for 20.5; but 64 x 4096 x 4096 14.9 for 10.1), and weights of odd rows go
  // there too (4 or 16 rows by 14336 of 4099 codes 16 and 19 us; a kernel that loads them into registers took 25 and 33).
  const bool rows = whole && (a->M <= 32 || (a->M <= kFewRows && (int64_t)a->N * products <= 8192));
  if (o.is("rows") ? whole && a->M <= kFewRows : rows && !o.tiles()) {
    q->kernel = kRows;
    return CMPEXT3_OK;
  }
  const double copies = products == 2 ? copy_us({&q->x, &q->w[0], &q->w[1]}, esz) : copy_us({&q->x, &q->w[0]}, esz);
  q->tile = plan_tiles(a->M, a->N, cdiv(a->K * (int64_t)esz, 128), products, 1, copies, true, true);
  if (q->tile.bm == 0) return CMPEXT3_OK;
  q->kernel = kTile;
  if (q->tile.bm > 64) {
    plan_copy(&q->x, esz, &q->ws_bytes);
    for (int i = 0; i < products; ++i) plan_copy(&q->w[i], esz, &q->ws_bytes);
  }
  q->partials_at = take(&q->ws_bytes, partial_bytes(q->tile, a->M, a->N, products, 1));
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
  p.out[0] = a->out;
  p.ldo[0] = a->out_row;
  p.out_dtype = a->out_dtype;
  p.pre[0] = a->gate_out;
  p.pre[1] = a->up_out;
  p.ld_pre = a->pre_row;
  p.pre_vec = a->pre_row % 4 == 0 && aligned(a->gate_out, 16) && aligned(a->up_out, 16);
  p.act = a->activation;
  p.M = a->M, p.N = a->N, p.K = a->K;
  p.batch = p.splits = 1;
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
  if (a->M * cdiv(a->N, 2048) * 256 > kMostThreads) return CMPEXT3_ERR_TOO_LARGE;
  return CMPEXT3_OK;
}

// Elements of a row of the held gradients: whole 16 bytes.
int64_t grad_pitch(int N) { return cdiv(N, 8) * 8; }

struct BackwardPlan {
  int64_t d_at[2], d_col_at[2];  // dgate and dup: bf16, or f16 for dx; f16 for the weights; -1: not needed
  int64_t row_at[2], col_at[2], most_at[2];  // f16: units and inverses of rows, of columns; their largest values
  GradUnits units;
  Operand w[2], x;  // [K, N] operands of the products: rows across k
  TilePlan dx, dw;
  int64_t partials_at, ws_bytes;
};

int plan_backward(const cmpext3_gated_backward_args* a, BackwardPlan* q) {
  const int st = check_gated_backward(a);
  if (st != CMPEXT3_OK) return st;
  *q = BackwardPlan{};
  const int64_t pitch = grad_pitch(a->N), held = (int64_t)a->M * pitch * 2;
  const bool f16 = a->dtype == CMPEXT3_F16;
  const void* dw[2] = {a->dw_gate, a->dw_up};
  for (int i = 0; i < 2; ++i) {
    q->d_at[i] = !f16 || a->dx != nullptr ? take(&q->ws_bytes, held) : -1;
    q->d_col_at[i] = f16 && dw[i] != nullptr ? take(&q->ws_bytes, held) : -1;
  }
  if (f16 && a->M > 0 && a->N > 0) {
    GradUnits& u = q->units;
    grad_blocks(a->M, a->N, &u);
    for (int i = 0; i < 2; ++i) {
      q->row_at[i] = take(&q->ws_bytes, 4 * (int64_t)a->M);
      q->col_at[i] = take(&q->ws_bytes, 4 * 2 * pitch);
    }
    q->most_at[0] = take(&q->ws_bytes, 4 * (int64_t)u.col_blocks * a->M);
    q->most_at[1] = take(&q->ws_bytes, 4 * (int64_t)u.row_blocks * 2 * pitch);
  }
  q->w[0] = Operand{a->w_gate, a->gate_row, a->N, a->K, -1, 0};
  q->w[1] = Operand{a->w_up, a->up_row, a->N, a->K, -1, 0};
  q->x = Operand{a->x, a->x_row, a->M, a->K, -1, 0};
  if (a->M == 0 || a->N == 0 || a->K == 0 || read_override().is("any64x64")) return CMPEXT3_OK;
  const int64_t batch = (a->dw_gate != nullptr) + (a->dw_up != nullptr);
  int64_t partials = 0;
  // the small tiles read 16 bytes of a row at least: of x and the weights, and of dgate's and dup's N
  const bool rows16 = a->K >= 8 && a->N >= 8;
  if (a->dx != nullptr) {
    q->dx = plan_tiles(a->M, a->K, 2 * cdiv(a->N, 64), 1, 1, copy_us({&q->w[0], &q->w[1]}, 2), rows16, false);
    if (q->dx.bm > 64)
      for (Operand& w : q->w) plan_copy(&w, 2, &q->ws_bytes);
    partials = partial_bytes(q->dx, a->M, a->K, 1, 1);
  }
  if (batch > 0) {
    q->dw = plan_tiles(a->N, a->K, cdiv(a->M, 64), 1, batch, copy_us({&q->x}, 2), rows16, false);
    if (q->dw.bm > 64) plan_copy(&q->x, 2, &q->ws_bytes);
    partials = std::max(partials, partial_bytes(q->dw, a->N, a->K, 1, batch));
  }
  q->partials_at = take(&q->ws_bytes, partials);
  return CMPEXT3_OK;
}

}  // namespace

extern "C" int cmpext3_quantize_int8(const cmpext3_quantize_int8_args* a, void* stream) {
  if (a == nullptr) return CMPEXT3_ERR_INVALID_ARG;
  if (!is16(a->dtype) && a->dtype != CMPEXT3_F32) return CMPEXT3_ERR_UNSUPPORTED;
  if (a->rows < 0 || a->cols < 0) return CMPEXT3_ERR_INVALID_ARG;
  if (a->rows == 0) return CMPEXT3_OK;
  if (a->rows > kMostThreads / 256 || a->cols > kMostSize) return CMPEXT3_ERR_TOO_LARGE;
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
  p.cols = p.written = a->cols;
  return (int)launch_quantize_int8(a->dtype, p, (hipStream_t)stream);
}

extern "C" int64_t cmpext3_projection_workspace_size(const cmpext3_projection_args* a) {
  ProjPlan q;
  const int st = plan_projection(a, &q);
  return st != CMPEXT3_OK ? st : q.ws_bytes;
}

extern "C" int cmpext3_projection(const cmpext3_projection_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  ProjPlan q;
  int st = plan_projection(a, &q);
  if (st == CMPEXT3_OK) st = check_workspace(q.ws_bytes, workspace, workspace_bytes);
  if (st != CMPEXT3_OK) return st;
  if (a->M == 0 || a->N == 0) return CMPEXT3_OK;
  const hipStream_t s = (hipStream_t)stream;
  const ProjMode mode = a->w_up != nullptr ? kProjGated : kProjPlain;
  ProjParams p = params_of(a);
  if (q.make_inside) return (int)launch_projection_rows_codes(a->x_dtype, mode, p, s);
  if (q.make) {
    QuantParams c{};
    c.x = a->x;
    c.ldx = a->x_row;
    c.codes = (int8_t*)workspace + q.codes_at;
    c.ldc = c.written = (int)q.x.ld;
    c.scale = (float*)((char*)workspace + q.scale_at);
    c.rows = a->M, c.cols = a->K;
    const hipError_t e = launch_quantize_int8(a->x_dtype, c, s);
    if (e != hipSuccess) return (int)e;
    q.x.p = p.a[0] = p.a[1] = c.codes;
    p.lda = c.ldc;
    p.a_scale = c.scale;
  }
  if (q.kernel == kAny) return (int)launch_projection_any(a->dtype, mode, false, false, p, s);
  if (q.kernel == kRows) return (int)launch_projection_rows(a->dtype, mode, p, s);
  const size_t esz = elem_size(a->dtype);
  const hipError_t e = run_copies({&q.x, &q.w[0], &q.w[1]}, esz, (char*)workspace, s);
  if (e != hipSuccess) return (int)e;
  p.a[0] = p.a[1] = q.x.p;
  p.lda = q.x.ld;
  for (int i = 0; i < 2; ++i) p.b[i] = q.w[i].p, p.ldb[i] = q.w[i].ld;
  if (q.tile.bm > 64) p.K = (int)(cdiv(a->K * (int64_t)esz, 16) * 16 / (int64_t)esz);  // copies hold zeros up to there
  ProjTileLaunch* launch = a->dtype == CMPEXT3_F16    ? launch_projection_tile_gated_f16
                           : a->dtype == CMPEXT3_BF16 ? launch_projection_tile_gated_bf16
                           : mode == kProjGated       ? launch_projection_tile_int8_gated
                                                      : launch_projection_tile_int8_plain;
  return (int)run_tiles(a->dtype, mode, launch, q.tile, p, (char*)workspace + q.partials_at, s);
}

extern "C" int cmpext3_projection_describe(const cmpext3_projection_args* a, char* buf, int buflen) {
  ProjPlan q;
  const int st = plan_projection(a, &q);
  if (st != CMPEXT3_OK) return st;
  if (buf == nullptr || buflen <= 0) return CMPEXT3_OK;
  if (a->M == 0 || a->N == 0)
    snprintf(buf, (size_t)buflen, "kernel=none");
  else if (q.kernel != kTile)
    snprintf(buf, (size_t)buflen, "kernel=%s%s", q.kernel == kRows ? "rows" : "any64x64", q.make_inside ? " codes=inside" : "");
  else
    snprintf(buf, (size_t)buflen, "kernel=%s%dx%d%s groups=%d splits=%d copies=%d", q.tile.bm == 64 ? "small" : "tile", q.tile.bm, q.tile.bn, q.tile.deep ? " ring=4" : "", q.tile.groups, q.tile.splits,
             (q.x.copy_at >= 0) + (q.w[0].copy_at >= 0) + (q.w[1].copy_at >= 0));
  return CMPEXT3_OK;
}

extern "C" int64_t cmpext3_gated_backward_workspace_size(const cmpext3_gated_backward_args* a) {
  BackwardPlan q;
  const int st = plan_backward(a, &q);
  return st != CMPEXT3_OK ? st : q.ws_bytes;
}

extern "C" int cmpext3_gated_backward(const cmpext3_gated_backward_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
  BackwardPlan q;
  int st = plan_backward(a, &q);
  if (st == CMPEXT3_OK) st = check_workspace(q.ws_bytes, workspace, workspace_bytes);
  if (st != CMPEXT3_OK) return st;
  const hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  const bool f16 = a->dtype == CMPEXT3_F16;
  const int64_t pitch = grad_pitch(a->N);
  auto at = [&](int64_t offset) -> char* { return offset >= 0 ? ws + offset : nullptr; };
  void* const d[2] = {at(q.d_at[0]), at(q.d_at[1])};
  void* const d_col[2] = {f16 ? at(q.d_col_at[0]) : d[0], f16 ? at(q.d_col_at[1]) : d[1]};
  const bool units = f16 && a->M > 0 && a->N > 0;
  GradUnits u = q.units;
  hipError_t e = hipSuccess;
  if (a->M > 0 && a->N > 0) {
    GatedGradParams g{};
    g.grad = a->grad_out;
    g.gate = a->gate;
    g.up = a->up;
    for (int i = 0; i < 2; ++i) g.d[i] = d[i], g.d_col[i] = f16 ? d_col[i] : nullptr;
    if (units) {
      u.row = (float*)at(q.row_at[0]), u.row_inverse = (float*)at(q.row_at[1]);
      u.col = (float*)at(q.col_at[0]), u.col_inverse = (float*)at(q.col_at[1]);
      u.row_most = (uint32_t*)at(q.most_at[0]), u.col_most = (uint32_t*)at(q.most_at[1]);
      g.units = u;
    }
    g.ld_grad = a->grad_row, g.ld_pre = a->pre_row, g.ld_d = pitch;
    g.act = a->activation;
    g.M = a->M, g.N = a->N;
    e = launch_gated_grad(a->dtype, g, s);
    if (e != hipSuccess) return (int)e;
  }
  e = run_copies({&q.w[0], &q.w[1], &q.x}, 2, ws, s);
  if (e != hipSuccess) return (int)e;
  ProjParams p{};
  p.out_dtype = a->dtype;
  p.lda = pitch;
  p.a[0] = d[0], p.a[1] = d[1];
  p.a_scale = units ? u.row_inverse : nullptr;
  p.batch = p.splits = 1;
  if (a->dx != nullptr && a->M > 0 && a->K > 0) {
    for (int i = 0; i < 2; ++i) p.b[i] = q.w[i].p, p.ldb[i] = q.w[i].ld;
    p.out[0] = a->dx;
    p.ldo[0] = a->dx_row;
    p.M = a->M, p.N = a->K, p.K = a->N;
    e = q.dx.bm == 0 ? launch_projection_any(a->dtype, kProjSum, false, true, p, s)
                     : run_tiles(a->dtype, kProjSum, f16 ? launch_projection_tile_sum_f16 : launch_projection_tile_sum_bf16, q.dx, p,
                                 ws + q.partials_at, s);
    if (e != hipSuccess) return (int)e;
  }
  // the weights' gradients that are asked for, as one batch
  p.batch = 0;
  void* dw[2] = {a->dw_gate, a->dw_up};
  const int64_t dw_row[2] = {a->dgate_row, a->dup_row};
  for (int i = 0; i < 2; ++i) {
    if (dw[i] == nullptr) continue;
    p.a[p.batch] = d_col[i];
    if (units && p.batch == 0) p.a_scale = u.col_inverse + i * (int64_t)a->N;
    p.out[p.batch] = dw[i];
    p.ldo[p.batch] = dw_row[i];
    ++p.batch;
  }
  if (p.batch == 0 || a->N == 0 || a->K == 0) return CMPEXT3_OK;
  p.b[0] = q.x.p, p.ldb[0] = q.x.ld;
  p.M = a->N, p.N = a->K, p.K = a->M;
  return (int)(q.dw.bm == 0 ? launch_projection_any(a->dtype, kProjPlain, true, true, p, s)
                            : run_tiles(a->dtype, kProjPlain, f16 ? launch_projection_tile_wgrad_f16 : launch_projection_tile_wgrad_bf16,
                                        q.dw, p, ws + q.partials_at, s));
}
