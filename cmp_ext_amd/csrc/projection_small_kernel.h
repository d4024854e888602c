// Products of the feed-forward operators in 64 x 64 tiles, for operands of any alignment and for few results: where
// the large tiles would leave CUs idle, or would need copies of their operands first.
//
// A workgroup of four waves, 32 x 32 results each.  A step of 128 bytes of k goes through registers, DEPTH steps
// ahead, into one of two LDS slots, so that one barrier a step is enough and several workgroups share a CU.
// Lanes load 16 bytes from any address: rows along k lie in LDS as the large tiles have them (lds_off128), rows
// across k (B as [K, N], A as [K, M]) as [k][64 columns] for the transposing reads (kn128_off).  Where 16 bytes
// would run past their row they are loaded from where they end with it, and shifted.  Rows past the last one
// are read as the last one (their results are not stored), steps of k past the end are zeros.
#pragma once

#include "projection_common.h"

namespace cmpext3 {

constexpr int kSmallTile = 64;

typedef u32x4 u32x4_any __attribute__((aligned(1)));

// v without its first `bytes` bytes (0 to 16), zeros behind.
__device__ __forceinline__ u32x4 drop_bytes(u32x4 v, int bytes) {
  unsigned __int128 x = __builtin_bit_cast(unsigned __int128, v);
  x = bytes >= 16 ? 0 : x >> (8 * bytes);
  return __builtin_bit_cast(u32x4, x);
}

// One operand's share of a thread: two 16-byte pieces of each step.
template <int ESZ, bool ACROSS>
struct SmallOperand {
  const char* row[2];  // along k: the piece's row; across: the operand's start
  int64_t ld;          // bytes of a row
  int64_t length;      // bytes of a row that are the operand's
  int K;
  uint32_t lds[2];
  int at[2];    // bytes within a row: along k, of the step; across, of the row
  int k[2];     // across: row of the step
  bool edge;    // across: the tile reaches past the last column

  // rows: of the operand along k, or its columns across it; first: the tile's first one
  __device__ __forceinline__ void init(const void* p, int64_t pitch, int rows, int first, int K_) {
    ld = pitch * ESZ;
    K = K_;
    edge = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = threadIdx.x + 256 * i, r = q >> 3, chunk = q & 7;
      if constexpr (ACROSS) {
        length = (int64_t)rows * ESZ;
        row[i] = (const char*)p;
        k[i] = r;
        at[i] = first * ESZ + 16 * chunk;  // 64 columns of 2 bytes: 128 bytes
        lds[i] = kn128_off(r, 16 * chunk);
        edge = first + kSmallTile > rows;
      } else {
        length = (int64_t)K * ESZ;
        row[i] = (const char*)p + (int64_t)min(first + r, rows - 1) * ld;
        k[i] = 0;
        at[i] = 16 * chunk;
        lds[i] = lds_off128(r, chunk);
      }
    }
  }
  // gated: rows 0..15 of every 32 of the tile are of the first weight, the others the same rows of the second
  __device__ __forceinline__ void init_pair(const ProjParams& p, int first) {
    static_assert(!ACROSS, "weights along k");
    K = p.K;
    length = (int64_t)K * ESZ;
    edge = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = threadIdx.x + 256 * i, r = q >> 3, chunk = q & 7;
      const bool second = (r >> 4) & 1;
      const int64_t n = min(first + (r >> 5) * 16 + (r & 15), p.N - 1);
      row[i] = (const char*)(second ? p.b[1] : p.b[0]) + n * (second ? p.ldb[1] : p.ldb[0]) * ESZ;
      k[i] = 0;
      at[i] = 16 * chunk;
      lds[i] = lds_off128(r, chunk);
    }
  }
  __device__ __forceinline__ void load(u32x4* v, int step) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (ACROSS) {
        const int64_t kk = min((int64_t)step * (128 / ESZ) + k[i], (int64_t)K - 1);
        v[i] = *(const u32x4_any*)(row[i] + kk * ld + min((int64_t)at[i], length - 16));
      } else {
        v[i] = *(const u32x4_any*)(row[i] + min((int64_t)step * 128 + at[i], length - 16));
      }
    }
  }
  // whether pieces of the step run past their row or the last k (the same for the whole workgroup)
  __device__ __forceinline__ bool cut(int step) const {
    return edge || (step + 1) * (int64_t)(128 / ESZ) > K;
  }
  template <bool CUT>
  __device__ __forceinline__ void store(unsigned char* slot, const u32x4* v, int step) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u32x4 x = v[i];
      if constexpr (CUT) {
        const int64_t from = (ACROSS ? 0 : (int64_t)step * 128) + at[i];
        x = drop_bytes(x, (int)min(max(from + 16 - length, (int64_t)0), (int64_t)16));
        if (ACROSS && (int64_t)step * (128 / ESZ) + k[i] >= K) x = u32x4{0, 0, 0, 0};
      }
      *(u32x4*)(slot + lds[i]) = x;
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

template <typename T, int MODE, bool AKM, bool BKN, int DEPTH, bool SPLITK>
__global__ void __launch_bounds__(256) projection_small_kernel(const ProjParams p) {
  using Acc = typename Prod<T>::Acc;
  constexpr bool GATED = MODE == kProjGated, SUM = MODE == kProjSum;
  constexpr int ESZ = sizeof(T), BK = 128 / ESZ;
  constexpr int COLS = GATED ? 32 : 64;  // of results
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2][2][kSmallTile * 128];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
    b[0].init_pair(p, n0);
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
  auto store = [&](int d, int kt) {  // both parts' rows lie alike
    const int step = SUM && first + kt >= part_steps ? first + kt - part_steps : first + kt;
    if (a[0].cut(step) || b[0].cut(step)) {
      a[0].template store<true>(smem[kt & 1][0], va[d], step);
      b[0].template store<true>(smem[kt & 1][1], vb[d], step);
    } else {
      a[0].template store<false>(smem[kt & 1][0], va[d], step);
      b[0].template store<false>(smem[kt & 1][1], vb[d], step);
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
  auto multiply = [&](int kt) {
    const unsigned char* ta = smem[kt & 1][0];
    const unsigned char* tb = smem[kt & 1][1];
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
  // past the end the last step is loaded again and not used: a load under a condition would make the compiler
  // wait for all that are on their way
  if (nk > 0) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      load(d, min(d, nk - 1));
      __builtin_amdgcn_sched_barrier(0);  // in this order, as the loop waits for them
    }
  }
  auto step = [&](int d, int kt, auto more) {
    store(d, kt);
    if constexpr (decltype(more)::value) load(d, min(kt + DEPTH, nk - 1));
    // this wave's part of the slot is written; every wave is past its reads of the slot before
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
    multiply(kt);
  };
  int kt = 0;
  for (; kt + DEPTH <= nk; kt += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) step(d, kt + d, std::true_type{});
  }
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d)
    if (kt + d < nk) step(d, kt + d, std::false_type{});

  // ---- acc[i][j][e]: row 16i + r16, B tile row 16j + 4G + e of the wave's block ----
  const int nw = n0 + (GATED ? wn / 2 : wn) + 4 * G;
  if constexpr (SPLITK) {
    constexpr int NP = GATED ? 2 : 1;
    uint32_t* part = (uint32_t*)p.partials + ((int64_t)ks * p.batch + bz) * NP * p.M * p.ld_part;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int64_t m = m0 + wm + 16 * (x >> 1) + r16;
      const int n = nw + (GATED ? 0 : 16 * (x & 1));
      if (m < p.M && n < p.N)
        *(u32x4*)(part + ((GATED ? (x & 1) * (int64_t)p.M : 0) + m) * p.ld_part + n) = __builtin_bit_cast(u32x4, acc[x >> 1][x & 1]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + wm + 16 * i + r16;
    if (m >= p.M) continue;
    const float as = ESZ == 1 ? p.a_scale[m] : 1.f;
    f32x4 v[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = nw + (GATED ? 0 : 16 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[j][e] = (float)acc[i][j][e];
        if (ESZ == 1) v[j][e] = v[j][e] * as * (n + e < p.N ? p.b_scale[GATED ? j : 0][n + e] : 0.f);
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
hipError_t launch_projection_small(const ProjParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)(p.batch * p.splits)), block(256);
  if (p.splits > 1) return launch_kernel((projection_small_kernel<T, MODE, AKM, BKN, 3, true>), grid, block, 0, s, p);
  return launch_kernel((projection_small_kernel<T, MODE, AKM, BKN, 3, false>), grid, block, 0, s, p);
}

}  // namespace cmpext3
