// The second launch of a product whose K was split: adds the splits' sums in their order and finishes
// the results.  Bound by reading the sums: splits x 4 bytes a result and product.
#include "projection_common.h"

namespace cmpext3 {
namespace {

template <typename T, int MODE>
__global__ void __launch_bounds__(256) projection_join_kernel(const ProjParams p) {
  using Acc = typename Prod<T>::Acc;
  constexpr int NP = MODE == kProjGated ? 2 : 1;
  const int bz = blockIdx.z;
  const int64_t per_row = p.ld_part / 4;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = at / per_row;
  const int n0 = (int)(at - m * per_row) * 4;
  if (m >= p.M || n0 >= p.N) return;
  // f16 gradients' units, whose inverse only they have
  const float unit = sizeof(T) != 1 && MODE == kProjPlain && p.a_scale != nullptr ? p.a_scale[bz * (int64_t)p.M + m] : 1.f;
  f32x4 v[NP];
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    Acc sum = Prod<T>::zero();
    const Acc* src = (const Acc*)p.partials + (((int64_t)bz * NP + q) * p.M + m) * per_row + n0 / 4;
    const int64_t stride = (int64_t)p.batch * NP * p.M * per_row;
    for (int s = 0; s < p.splits; ++s) sum += src[s * stride];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[q][e] = (float)sum[e];
      if (sizeof(T) == 1 && n0 + e < p.N) v[q][e] = RowScaled(p.a_scale[m])(v[q][e], p.b_scale[q][n0 + e]);
      if (sizeof(T) != 1 && MODE == kProjPlain) v[q][e] *= unit;
    }
  }
  f32x4 y = v[0];
  if constexpr (MODE == kProjGated) {
    with_act(p.act, [&](auto act) {
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = act_value<decltype(act)::value>(v[0][e]) * v[1][e];
    });
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n0 + e >= p.N) break;
    if (MODE == kProjGated && p.pre[0] != nullptr) {
      p.pre[0][m * p.ld_pre + n0 + e] = v[0][e];
      p.pre[NP - 1][m * p.ld_pre + n0 + e] = v[NP - 1][e];
    }
    float r = y[e];
    if (MODE == kProjPlain && p.bias != nullptr) r += load_elem(p.bias, n0 + e, p.out_dtype);
    store_elem(p.out[bz], m * p.ldo[bz] + n0 + e, p.out_dtype, r);
  }
}

template <typename T>
hipError_t launch(ProjMode mode, const ProjParams& p, dim3 grid, hipStream_t s) {
  if (mode == kProjGated) return launch_kernel((projection_join_kernel<T, kProjGated>), grid, dim3(256), 0, s, p);
  return launch_kernel((projection_join_kernel<T, kProjPlain>), grid, dim3(256), 0, s, p);
}

}  // namespace

hipError_t launch_projection_join(int dtype, ProjMode mode, const ProjParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.M * (p.ld_part / 4) + 255) / 256), 1, (unsigned)p.batch);
  return dtype == kI8 ? launch<int8_t>(mode, p, grid, s) : launch<float>(mode, p, grid, s);
}

}  // namespace cmpext3
