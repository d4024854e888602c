// Products of the feed-forward operators in 64 x 64 tiles, for operands of any alignment and for few results: where
// the large tiles would leave CUs idle, or would need copies of their operands first.
//
// A workgroup of four waves, 32 x 32 results each.  A step of 128 bytes of k goes through registers, DEPTH steps
// ahead, into one of two LDS slots, so that one barrier a step is enough and several workgroups share a CU.
// Lanes load 16 bytes from any address: rows along k lie in LDS as the large tiles have them (lds_off128), rows
// across k (B as [K, N], A as [K, M]) as [k][64 columns] for the transposing reads (kn128_off).  Where 16 bytes
// would run past their row they are loaded from where they end with it, and shifted.  Rows past the last one
// are read as the last one (their results are not stored), steps of k past the end are zeros.
//
// What bounds it: the chain of a step (0.2 to 0.28 us where a workgroup is alone on its CU: store, barrier, read,
// multiply), and LDS at full CUs (0.65 us a step of three workgroups).  MI355X: codes x[333, 2050] by 1001 rows 10.7 us, gated
// fp16 x[77, 1001], two of 2731, 10.2, gated codes x[100, 1000], two of 4099, 8.5; 128 x 128 tiles on copies 18.7, 20 and 28.
#pragma once

#include "projection_common.h"

namespace cmpext3 {

constexpr int kSmallTile = 64;

// One operand's share of a thread: two 16-byte pieces of each step, in rows r and r + 32 of its tile (of the
// step, across).  Addresses are a scalar base that moves with the steps and 32-bit offsets within the tile.
template <int ESZ, bool ACROSS>
struct SmallOperand {
  const char* base;  // along k: the tile's first row; across: the operand
  int64_t ld;        // bytes of a row
  int length, K;     // bytes of a row that are the operand's; its k
  uint32_t off[2];   // along k: of the pieces' rows
  int r, at;         // across: row of the step; bytes within a row: along k, of the step
  uint32_t lds;
  bool edge;  // across: the tile reaches past the last column

  __device__ __forceinline__ void place(const char* first_row, int64_t pitch, int length_, int K_) {
    base = first_row;
    ld = pitch * ESZ;
    length = length_;
    K = K_;
    r = (threadIdx.x % 256) >> 3;
    at = 16 * (threadIdx.x & 7);
    lds = ACROSS ? kn128_off(r, at) : lds_off128(r, at >> 4);  // 32 rows on: 4096 bytes
    edge = false;
  }
  // rows: of the operand along k, or its columns across it; first: the tile's first one
  __device__ __forceinline__ void init(const void* p, int64_t pitch, int rows, int first, int K_) {
    if constexpr (ACROSS) {
      place((const char*)p, pitch, rows * ESZ, K_);
      at += first * ESZ;  // 64 columns of 2 bytes: 128 bytes
      edge = first + kSmallTile > rows;
    } else {
      place((const char*)p + first * (pitch * ESZ), pitch, K_ * ESZ, K_);
#pragma unroll
      for (int i = 0; i < 2; ++i) off[i] = (uint32_t)(min(r + 32 * i, rows - 1 - first) * ld);
    }
  }
  // gated: rows 0..15 of every 32 of the tile are of the first weight (waves 0 and 1), the others the same rows of
  // the second
  __device__ __forceinline__ void init_pair(const ProjParams& p, int first, int wave) {
    static_assert(!ACROSS, "weights along k");
    const int which = wave >> 1;
    place((const char*)p.b[which] + first * (p.ldb[which] * ESZ), p.ldb[which], p.K * ESZ, p.K);
#pragma unroll
    for (int i = 0; i < 2; ++i) off[i] = (uint32_t)(min((r & 15) + 16 * i, p.N - 1 - first) * ld);
  }
  __device__ __forceinline__ void load(u32x4* v, int step) const {
    if constexpr (ACROSS) {
      const int k0 = step * (128 / ESZ);
      const char* row0 = base + k0 * ld;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        v[i] = *(const u32x4_any*)(row0 + (uint32_t)(min(r + 32 * i, K - 1 - k0) * (int)ld + min(at, length - 16)));
    } else {
      const uint32_t from = (uint32_t)min(step * 128 + at, length - 16);
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] = *(const u32x4_any*)(base + (off[i] + from));
    }
  }
  // whether pieces of the step run past their row or the last k (the same for the whole workgroup)
  __device__ __forceinline__ bool cut(int step) const { return edge || (step + 1) * (128 / ESZ) > K; }
  template <bool CUT>
  __device__ __forceinline__ void store(unsigned char* slot, const u32x4* v, int step) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u32x4 x = v[i];
      if constexpr (CUT) {
        x = drop_bytes(x, min(max((ACROSS ? 0 : step * 128) + at + 16 - length, 0), 16));
        if (ACROSS && step * (128 / ESZ) + r + 32 * i >= K) x = u32x4{0, 0, 0, 0};
      }
      *(u32x4*)(slot + lds + 4096 * i) = x;
    }
  }
};

// Four results of a row, as far as the columns go.
__device__ __forceinline__ void store_four(void* out, int64_t row_at, int n, int N, int dtype, f32x4 y) {
  typedef f32x4 f32x4_e __attribute__((aligned(4)));
  typedef u32x2 u32x2_e __attribute__((aligned(2)));
  if (n + 4 <= N) {
    if (dtype == kF32)
      *(f32x4_e*)((float*)out + row_at + n) = y;
    else
      *(u32x2_e*)((uint16_t*)out + row_at + n) =
          dtype == kF16 ? u32x2{pack2<_Float16>(y[0], y[1]), pack2<_Float16>(y[2], y[3])} : u32x2{pack2<__bf16>(y[0], y[1]), pack2<__bf16>(y[2], y[3])};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < N) store_elem(out, row_at + n + e, dtype, y[e]);
}

// GROUPS: of four waves, which take a tile's steps in turn; their sums are added at the end.
template <typename T, int MODE, bool AKM, bool BKN, int DEPTH, int GROUPS, bool SPLITK>
__global__ void __launch_bounds__(256 * GROUPS) projection_small_kernel(const ProjParams p) {
  using Acc = typename Prod<T>::Acc;
  constexpr bool GATED = MODE == kProjGated, SUM = MODE == kProjSum;
  constexpr int ESZ = sizeof(T), BK = 128 / ESZ;
  constexpr int COLS = GATED ? 32 : 64;  // of results
  __shared__ __attribute__((aligned(1024))) unsigned char slots[GROUPS][2][2][kSmallTile * 128];
  const int lane = threadIdx.x & 63;
  const int group = GROUPS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  auto& smem = slots[group];
  const int r16 = lane & 15, G = lane >> 4;
  const int wm = 32 * (wave >> 1), wn = 32 * (wave & 1);
  int tm, tn, bzi;
  tile_coords(blockIdx.x, blockIdx.z, gridDim.z, p.tiles_m, p.tiles_n, p.group_m, tm, tn, bzi);
  const int m0 = tm * kSmallTile, n0 = tn * COLS;
  const int ks = SPLITK ? bzi % p.splits : 0;
  const int bz = SPLITK ? bzi / p.splits : bzi;
  const int part_steps = (p.K + BK - 1) / BK;
  const int all_steps = SUM ? 2 * part_steps : part_steps;
  const int first = SPLITK ? ks * p.ksplit : 0;
  const int nk = SPLITK ? min(all_steps - first, p.ksplit) : all_steps;

  SmallOperand<ESZ, AKM> a[SUM ? 2 : 1];
  SmallOperand<ESZ, BKN> b[SUM ? 2 : 1];
  a[0].init(p.a[SUM ? 0 : bz], p.lda, p.M, m0, p.K);
  if constexpr (GATED)
    b[0].init_pair(p, n0, wave);
  else
    b[0].init(p.b[0], p.ldb[0], p.N, n0, p.K);
  if constexpr (SUM) {
    a[1].init(p.a[1], p.lda, p.M, m0, p.K);
    b[1].init(p.b[1], p.ldb[1], p.N, n0, p.K);
  }
  u32x4 va[DEPTH][2], vb[DEPTH][2];
  auto load = [&](int d, int kt) {
    const int step = first + kt;
    if (SUM && step >= part_steps) {
      a[SUM ? 1 : 0].load(va[d], step - part_steps);
      b[SUM ? 1 : 0].load(vb[d], step - part_steps);
    } else {
      a[0].load(va[d], step);
      b[0].load(vb[d], step);
    }
  };
  auto store = [&](int d, int r) {  // both parts' rows lie alike
    const int kt = GROUPS * r + group;
    const int step = SUM && first + kt >= part_steps ? first + kt - part_steps : first + kt;
    if (a[0].cut(step) || b[0].cut(step)) {
      a[0].template store<true>(smem[r & 1][0], va[d], step);
      b[0].template store<true>(smem[r & 1][1], vb[d], step);
    } else {
      a[0].template store<false>(smem[r & 1][0], va[d], step);
      b[0].template store<false>(smem[r & 1][1], vb[d], step);
    }
  };

  // fragment addresses, as in the large tiles
  const int kr = 8 * G + (r16 >> 2);
  uint32_t fa_off[2], fb_off[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    fa_off[i] = AKM ? kn128_off(kr, (wm + 16 * i + 4 * (r16 & 3)) * 2) : lds_off128(wm + r16, 4 * i + G);
    fb_off[i] = BKN ? kn128_off(kr, (wn + 16 * i + 4 * (r16 & 3)) * 2) : lds_off128(wn + r16, 4 * i + G);
  }
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  auto fragment = [&](const unsigned char* tile, const uint32_t* off, auto across, int s, int i) {
    if constexpr (decltype(across)::value) {
      u32x4 f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // rows + 4 and + 32 change no term of the swizzle but (k / 2) % 2, which + 4 leaves too
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (__attribute__((address_space(3))) s16x4*)(tile + off[i] + (32 * s + 4 * half) * 128)));
        f[2 * half] = v.x;
        f[2 * half + 1] = v.y;
      }
      return f;
    } else {
      return *(const u32x4*)(tile + off[s] + i * 2048);
    }
  };
  Acc acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = Prod<T>::zero();
  auto multiply = [&](int r) {
    const unsigned char* ta = smem[r & 1][0];
    const unsigned char* tb = smem[r & 1][1];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = fragment(ta, fa_off, std::integral_constant<bool, AKM>{}, s, i);
        fb[i] = fragment(tb, fb_off, std::integral_constant<bool, BKN>{}, s, i);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = Prod<T>::mma(fb[i & 1], fa[i >> 1], acc[i >> 1][i & 1]);
    }
  };
  // Round r is step GROUPS r + group.  Past the end the last step is loaded again and not used: a load under a
  // condition would make the compiler wait for all that are on their way.
  auto load_round = [&](int d, int r) { load(d, min(GROUPS * r + group, nk - 1)); };
  if (nk > 0) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      load_round(d, d);
      __builtin_amdgcn_sched_barrier(0);  // in this order, as the loop waits for them
    }
  }
  auto fence = [] {
    // this wave's part of the slot is written; every wave is past its reads of the slot before
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
  };
  const int whole = nk / GROUPS, rounds = (nk + GROUPS - 1) / GROUPS;  // whole: every group has a step
  int r = 0;
  for (; r + DEPTH <= whole; r += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      store(d, r + d);
      load_round(d, r + d + DEPTH);
      fence();
      multiply(r + d);
    }
  }
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) {
    if (r + d >= rounds) break;
    const bool mine = GROUPS * (r + d) + group < nk;
    if (mine) store(d, r + d);
    fence();
    if (mine) multiply(r + d);
  }

  // ---- sums of the groups, in their order: group g then holds rows 16g .. of the wave's block ----
  static_assert(GROUPS <= 2, "a group for each of the wave's two row blocks");
  constexpr int I = GROUPS > 1 ? 1 : 2;  // row blocks that a group finishes
  if constexpr (GROUPS > 1) {
    Acc* sums = (Acc*)slots;  // [group][block][wave][lane]
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 4; ++x) sums[((group * 4 + x) * 4 + wave) * 64 + lane] = acc[x >> 1][x & 1];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      Acc sum = sums[((2 * group + j) * 4 + wave) * 64 + lane];
#pragma unroll
      for (int g = 1; g < GROUPS; ++g) sum += sums[((g * 4 + 2 * group + j) * 4 + wave) * 64 + lane];
      acc[0][j] = sum;
    }
  }
  const int i0 = GROUPS > 1 ? group : 0;

  // ---- acc[i][j][e]: row 16i + r16, B tile row 16j + 4G + e of the wave's block ----
  const int nw = n0 + (GATED ? wn / 2 : wn) + 4 * G;
  if constexpr (SPLITK) {
    constexpr int NP = GATED ? 2 : 1;
    uint32_t* part = (uint32_t*)p.partials + ((int64_t)ks * p.batch + bz) * NP * p.M * p.ld_part;
#pragma unroll
    for (int x = 0; x < 2 * I; ++x) {
      const int64_t m = m0 + wm + 16 * (i0 + (x >> 1)) + r16;
      const int n = nw + (GATED ? 0 : 16 * (x & 1));
      if (m < p.M && n < p.N)
        *(u32x4*)(part + ((GATED ? (x & 1) * (int64_t)p.M : 0) + m) * p.ld_part + n) = __builtin_bit_cast(u32x4, acc[x >> 1][x & 1]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int64_t m = m0 + wm + 16 * (i0 + i) + r16;
    if (m >= p.M) continue;
    const float as = ESZ == 1 ? p.a_scale[m] : row_unit<T, MODE>(p, bz, m);
    const RowScaled scaled(as);
    f32x4 v[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = nw + (GATED ? 0 : 16 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[j][e] = (float)acc[i][j][e];
        if (ESZ != 1) v[j][e] *= as;
        if (ESZ == 1) v[j][e] = scaled(v[j][e], n + e < p.N ? p.b_scale[GATED ? j : 0][n + e] : 0.f);
        if (!GATED && ESZ == 1 && p.bias != nullptr && n + e < p.N) v[j][e] += load_elem(p.bias, n + e, p.out_dtype);
      }
    }
    if constexpr (GATED) {
      if (nw >= p.N) continue;
      if (p.pre[0] != nullptr) {
        store_four(p.pre[0], m * p.ld_pre, nw, p.N, kF32, v[0]);
        store_four(p.pre[1], m * p.ld_pre, nw, p.N, kF32, v[1]);
      }
      f32x4 y;
      with_act(p.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = act_value<decltype(act)::value>(v[0][e]) * v[1][e];
      });
      store_four(p.out[0], m * p.ldo[0], nw, p.N, p.out_dtype, y);
    } else {
      const int which = SUM ? 0 : bz;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (nw + 16 * j < p.N) store_four(p.out[which], m * p.ldo[which], nw + 16 * j, p.N, p.out_dtype, v[j]);
    }
  }
}

template <typename T, int MODE, bool AKM, bool BKN>
hipError_t launch_projection_small(const ProjParams& p, int groups, hipStream_t s) {
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)(p.batch * p.splits)), block(256 * groups);
  if (p.splits > 1) {
    if (groups == 2) return launch_kernel((projection_small_kernel<T, MODE, AKM, BKN, 3, 2, true>), grid, block, 0, s, p);
    return launch_kernel((projection_small_kernel<T, MODE, AKM, BKN, 3, 1, true>), grid, block, 0, s, p);
  }
  if (groups == 2) return launch_kernel((projection_small_kernel<T, MODE, AKM, BKN, 3, 2, false>), grid, block, 0, s, p);
  return launch_kernel((projection_small_kernel<T, MODE, AKM, BKN, 3, 1, false>), grid, block, 0, s, p);
}

}  // namespace cmpext3
