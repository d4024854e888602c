// Tiled products of the feed-forward operators on the matrix cores: 16-bit floats or 8-bit codes,
// one product or the two of a gated block, operands along k or across it.
//
// The main loop is that of the f16/bf16 tiles of plain products (tile16_kernel.h): K steps of 128
// bytes (64 16-bit elements, 128 codes) go global -> LDS by LDS-DMA into a ring, one barrier a step, and
// fragment reads and DMA pieces spread over the matrix instructions.  What differs:
//   * Codes take the same LDS layout: a fragment is 16 bytes of a row whatever they hold, and
//     v_mfma_i32_16x16x64_i8 takes twice the k of the 16-bit instruction from it in the same time.
//   * Gated: the B tile holds 16 rows of w_gate, the same 16 of w_up, and so on, so that a wave's
//     neighbouring accumulator blocks are both products of the same results: the activation and the
//     product happen in registers and only the result is stored (and, for a backward pass, both
//     products).
//   * Sum (the gradient of x): K runs through dgate w_gate, then dup w_up, in one sum.
//   * A across k (weight gradients, dgate^T x): [k][m] rows in LDS, read by the transposing
//     reads that B as [K, N] has there.
//   * f16 gradients: a row's sums times what undoes the unit that its operand was held in (gated_grad.hip).
//
// What bounds it at prompts and training batches: the board's power limit, as for the plain products.  MI355X, 256 x
// 256 tiles: gated bf16 4096 x 4096, two of 14336: 650 us, 1.48 PFLOP/s; dx 4096 x 28672 x 4096 650, dw 2 x 14336 x
// 4096 x 4096 681 (1.41 PFLOP/s); codes, 4096 x 14336 x 4096: 163, 2.95 POP/s, gated 2048 x 4096, two of 11008: 149.
// Both products stored in fp32 for the backward pass (470 MB more, which every CU stores at the end of its tile, all at
// once) cost some 100 us of the first.
#pragma once

#include "projection_common.h"

namespace cmpext3 {

// NSA, NSB: ring slots of A and of B, a step each.
template <int BM, int BN, bool AKM, bool BKN, int WM, int WN, int NSA, int NSB>
struct ProjTileShape {
  static constexpr int ROW = 128;  // bytes of k of a step
  static constexpr int NW = WM * WN;
  static constexpr int WTM = BM / WM, WTN = BN / WN;
  static constexpr int FM = WTM / 16, FN = WTN / 16;
  static constexpr int A_PITCH = AKM ? BM * 2 : ROW, B_PITCH = BKN ? BN * 2 : ROW;
  static constexpr int A_BYTES = BM * ROW, B_BYTES = BN * ROW;  // 64 k either way
  static constexpr int B_REGION = NSA * A_BYTES;
  static constexpr int LDS = NSA * A_BYTES + NSB * B_BYTES;
  static constexpr int A_DMA = A_BYTES / 1024 / NW, B_DMA = B_BYTES / 1024 / NW;
  static constexpr int DMA = A_DMA + B_DMA;
  static_assert(WTM % 16 == 0 && WTN % 32 == 0, "16-row blocks, pairs of 16-column blocks");
  static_assert(A_BYTES % (1024 * NW) == 0 && B_BYTES % (1024 * NW) == 0, "whole DMA loads per wave");
  static_assert(B_DMA % 4 == 0 || B_DMA == 2, "pairs of a wave's loads alternate between both weights, or the waves do");
  static_assert(LDS <= 160 * 1024, "LDS budget");
  static_assert(NSA >= 2 && NSB >= 2 && NSA * A_DMA + NSB * B_DMA - DMA <= 63, "vmcnt range");
  // offsets of a slot's reads are immediates up to 64 KiB; third slots of 32 KiB have a second base
  static_assert((NSA == 3 || (NSA - 1) * A_BYTES + (AKM ? 36 * A_PITCH : (FM - 1) * 2048) <= 65535) &&
                    (NSB == 3 || (NSB - 1) * B_BYTES + (BKN ? 36 * B_PITCH : (FN - 1) * 2048) <= 65535),
                "LDS offsets");
};

// O: the output's type.  KCHECK: K (of every part and split) is no multiple of a step.  SPLITK: grid.z =
// batch * splits; a workgroup stores its sums into p.partials.
template <typename T, typename O, int MODE, bool AKM, bool BKN, int BM, int BN, int WM, int WN, int MINB, int NSA, int NSB, bool KCHECK, bool SPLITK>
__global__ void __launch_bounds__(64 * WM * WN, MINB) projection_tile_kernel(const ProjParams p) {
  using S = ProjTileShape<BM, BN, AKM, BKN, WM, WN, NSA, NSB>;
  using Acc = typename Prod<T>::Acc;
  constexpr int FM = S::FM, FN = S::FN;
  constexpr bool GATED = MODE == kProjGated, SUM = MODE == kProjSum, CODES = sizeof(T) == 1;
  constexpr int E16 = 16 / sizeof(T);          // elements of a 16-byte piece
  constexpr int BK = S::ROW / sizeof(T);       // k of a step
  constexpr int OBN = GATED ? BN / 2 : BN;     // columns of results
  static_assert(!(CODES && (AKM || BKN)), "transposing reads are of 16-bit elements");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[S::LDS];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int tm, tn, bzi;
  tile_coords(blockIdx.x, blockIdx.z, gridDim.z, p.tiles_m, p.tiles_n, p.group_m, tm, tn, bzi);
  const int m0 = tm * BM, n0 = tn * OBN;
  const int M = p.M, N = p.N;
  const int ks = SPLITK ? bzi % p.splits : 0;
  const int bz = SPLITK ? bzi / p.splits : bzi;
  // steps of the whole sum (SUM: of both parts, one after the other) and this workgroup's range of them
  const int part_steps = (p.K + BK - 1) / BK;
  const int all_steps = SUM ? 2 * part_steps : part_steps;
  const int first = SPLITK ? ks * p.ksplit : 0;
  const int nk = SPLITK ? min(all_steps - first, p.ksplit) : all_steps;
  const int64_t lda = p.lda;
  const T* Abase[2];
  const T* Bbase[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    Abase[i] = (const T*)p.a[SUM ? i : bz] + (AKM ? (int64_t)m0 : (int64_t)m0 * lda);
    Bbase[i] = (const T*)p.b[i] + (BKN ? (int64_t)n0 : (int64_t)n0 * p.ldb[i]);
  }

  // ---- per-lane DMA sources, relative to the step's first k; rows past the matrix are out of range ----
  uint32_t a_off[S::A_DMA];
  int a_kx[S::A_DMA];
#pragma unroll
  for (int i = 0; i < S::A_DMA; ++i) {
    if constexpr (AKM) {
      int k, m;
      dma_kn_geom(wave * S::A_DMA + i, lane, S::A_PITCH, k, m);
      a_off[i] = m0 + m < M ? (uint32_t)(k * lda + m) * (uint32_t)sizeof(T) : kBufOOB;
      a_kx[i] = k;
    } else {
      int row, chunk;
      dma128_geom(wave * S::A_DMA + i, lane, row, chunk);
      a_off[i] = m0 + row < M ? (uint32_t)(row * lda + E16 * chunk) * (uint32_t)sizeof(T) : kBufOOB;
      a_kx[i] = E16 * chunk;
    }
  }
  uint32_t b_off[S::B_DMA];
  int b_kx[S::B_DMA];
#pragma unroll
  for (int i = 0; i < S::B_DMA; ++i) {
    if constexpr (BKN) {
      int k, n;
      dma_kn_geom(wave * S::B_DMA + i, lane, S::B_PITCH, k, n);
      b_off[i] = n0 + n < N ? (uint32_t)(k * p.ldb[0] + n) * (uint32_t)sizeof(T) : kBufOOB;
      b_kx[i] = k;
    } else {
      int row, chunk;
      dma128_geom(wave * S::B_DMA + i, lane, row, chunk);
      // gated: rows 0..15 of every 32 are of w_gate, the others the same rows of w_up
      const int col = GATED ? (row >> 5) * 16 + (row & 15) : row;
      const int64_t ldb = p.ldb[GATED ? (S::B_DMA == 2 ? wave & 1 : (i >> 1) & 1) : 0];
      b_off[i] = n0 + col < N ? (uint32_t)(col * ldb + E16 * chunk) * (uint32_t)sizeof(T) : kBufOOB;
      b_kx[i] = E16 * chunk;
    }
  }
  // SUM: both weights' pitches may differ, which per-lane offsets (made with the first's) leave to a
  // second set; a step of the second part takes those
  uint32_t b_off1[SUM ? S::B_DMA : 1];
  if constexpr (SUM) {
#pragma unroll
    for (int i = 0; i < S::B_DMA; ++i) {
      int k, n;
      dma_kn_geom(wave * S::B_DMA + i, lane, S::B_PITCH, k, n);
      b_off1[i] = n0 + n < N ? (uint32_t)(k * p.ldb[1] + n) * (uint32_t)sizeof(T) : kBufOOB;
    }
  }
  const uint32_t lds_a = lds_addr(smem) + (uint32_t)(wave * S::A_DMA * 1024);
  const uint32_t lds_b = lds_addr(smem) + (uint32_t)(S::B_REGION + wave * S::B_DMA * 1024);
  // gated: the weight that a wave's loads 0 and 1, and 2 and 3, are of
  i32x4 rsrc_pair[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    rsrc_pair[i] = make_rsrc_sgpr(Bbase[S::B_DMA == 2 ? wave & 1 : i]);
    rsrc_pair[i][0] = __builtin_amdgcn_readfirstlane(rsrc_pair[i][0]);
    rsrc_pair[i][1] = __builtin_amdgcn_readfirstlane(rsrc_pair[i][1]);
  }
  // LDS-DMA load d (A pieces first, then B) of step kt into ring slot `slot`.  Operands along k keep a
  // descriptor at the tile's base and advance through the scalar offset, operands across it get one per step;
  // a step past the end loads through a descriptor of no records (zeros, no memory read).
  auto dma_piece = [&](int kt, auto slotc, auto dc) {
    constexpr int slot = decltype(slotc)::value, d = decltype(dc)::value;
    const bool live = kt < nk;
    const int step = first + kt;
    const bool second = SUM && step >= part_steps;
    const int k0 = (second ? step - part_steps : step) * BK;
    if constexpr (d < S::A_DMA) {
      constexpr uint32_t dst = (uint32_t)(slot * S::A_BYTES + d * 1024);
      const uint32_t voff = !KCHECK || a_kx[d] < p.K - k0 ? a_off[d] : kBufOOB;
      const T* base = second ? Abase[1] : Abase[0];
      i32x4 r = make_rsrc_sgpr(AKM ? base + (int64_t)(live ? k0 : 0) * lda : base);
      r[2] = live ? (int)kBufRecords : 0;
      dma_load16_m0(r, voff, AKM ? 0u : (uint32_t)k0 * (uint32_t)sizeof(T), lds_a, std::integral_constant<uint32_t, dst>{});
    } else {
      constexpr int i = d - S::A_DMA;
      constexpr uint32_t dst = (uint32_t)(slot * S::B_BYTES + i * 1024);
      const uint32_t in = SUM && second ? b_off1[SUM ? i : 0] : b_off[i];
      const uint32_t voff = !KCHECK || b_kx[i] < p.K - k0 ? in : kBufOOB;
      i32x4 r;
      if constexpr (GATED) {
        r = rsrc_pair[(i >> 1) & 1];
      } else {
        const T* base = second ? Bbase[1] : Bbase[0];
        r = make_rsrc_sgpr(BKN ? base + (int64_t)(live ? k0 : 0) * (second ? p.ldb[1] : p.ldb[0]) : base);
      }
      r[2] = live ? (int)kBufRecords : 0;
      dma_load16_m0(r, voff, BKN ? 0u : (uint32_t)k0 * (uint32_t)sizeof(T), lds_b, std::integral_constant<uint32_t, dst>{});
    }
  };

  // ---- fragment addresses: lane (r16 = lane % 16, G = lane / 16) supplies row (column) r16 and bytes
  // 16G .. 16G+15 of a 64-byte sub-step ----
  const int r16 = lane & 15, G = lane >> 4;
  uint32_t fa_off[AKM ? FM : 2], fb_off[BKN ? FN : 2];
  // Across k: lanes of group G point at k row 8G + r16/4, columns 16i + 4(r16%4) of the wave's block; a
  // transposing read hands lane r16 column 16i + r16 at four consecutive k
  const int kr = 8 * G + (r16 >> 2);
  if constexpr (AKM) {
#pragma unroll
    for (int i = 0; i < FM; ++i) fa_off[i] = kn_off(kr, S::A_PITCH, (wm * S::WTM + 16 * i + 4 * (r16 & 3)) * 2);
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s) fa_off[s] = lds_off128(wm * S::WTM + r16, 4 * s + G);
  }
  if constexpr (BKN) {
#pragma unroll
    for (int j = 0; j < FN; ++j) fb_off[j] = S::B_REGION + kn_off(kr, S::B_PITCH, (wn * S::WTN + 16 * j + 4 * (r16 & 3)) * 2);
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s) fb_off[s] = S::B_REGION + lds_off128(wn * S::WTN + r16, 4 * s + G);
  }

  Acc acc[FM][FN];
  static_for<FM * FN>([&](auto xc) { acc[decltype(xc)::value / FN][decltype(xc)::value % FN] = Prod<T>::zero(); });

  typedef short s16x4 __attribute__((ext_vector_type(4)));
  u32x4 fa[2][FM], fb[2][FN];
  auto read_tr = [&](const unsigned char* q) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)q));
  };
  // LDS read r of sub-step s of a step's slot into fragment buffer buf
  constexpr int RA = (AKM ? 2 : 1) * FM, RD = RA + (BKN ? 2 : 1) * FN;
  auto read_one = [&](auto slotac, auto slotbc, int s, int buf, auto rc) {
    constexpr int r = decltype(rc)::value;
    const unsigned char* sa = smem + decltype(slotac)::value * S::A_BYTES;
    const unsigned char* sb = smem + decltype(slotbc)::value * S::B_BYTES;  // fb_off includes the B region's start
    if constexpr (r < RA && AKM) {
      constexpr int i = r >> 1, half = r & 1;
      const u32x2 v = read_tr(sa + fa_off[i] + (32 * s + 4 * half) * S::A_PITCH);
      fa[buf][i][2 * half] = v.x;
      fa[buf][i][2 * half + 1] = v.y;
    } else if constexpr (r < RA) {
      fa[buf][r] = *(const u32x4*)(sa + fa_off[s] + r * 16 * S::ROW);
    } else if constexpr (BKN) {
      constexpr int j = (r - RA) >> 1, half = (r - RA) & 1;
      const u32x2 v = read_tr(sb + fb_off[j] + (32 * s + 4 * half) * S::B_PITCH);
      fb[buf][j][2 * half] = v.x;
      fb[buf][j][2 * half + 1] = v.y;
    } else {
      constexpr int j = r - RA;
      fb[buf][j] = *(const u32x4*)(sb + fb_off[s] + j * 16 * S::ROW);
    }
  };
  // One sub-step of products on fragment buffer BUF; product x also issues its share of the reads of
  // sub-step RS of ring slots RA and RB into the other buffer and of ND DMA pieces.
  constexpr int X = FM * FN;
  auto substep = [&](auto bufc, auto rac, auto rbc, int rs, auto ndc, auto&& piece) {
    constexpr int buf = decltype(bufc)::value, nd = decltype(ndc)::value;
    static_for<X>([&](auto xc) {
      constexpr int x = decltype(xc)::value;
      constexpr int i = x / FN, j = x % FN;
      acc[i][j] = Prod<T>::mma(fb[buf][j], fa[buf][i], acc[i][j]);
      static_for<RD>([&](auto rc) {
        if constexpr (decltype(rc)::value * X / RD == x) read_one(rac, rbc, rs, buf ^ 1, rc);
      });
      static_for<nd>([&](auto dc) {
        if constexpr (decltype(dc)::value * X / nd == x) piece(dc);
      });
      __builtin_amdgcn_sched_barrier(0);  // keep the slots in this order
    });
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  using DA = std::integral_constant<int, S::DMA>;
  // Step kt, in every ring: all reads of its slots are issued by the end of the first sub-step, so that one
  // barrier both frees them and certifies the next step's data.
  if constexpr (NSA != NSB) {
    // One operand has a slot more, and a step more to arrive: its step kt + 3 is loaded behind the other's kt + 2, so
    // that it is what may be on its way at the next barrier.
    static_assert(NSA + NSB == 5, "rings of two and three steps");
    constexpr bool A_MORE = NSA == 3;
    constexpr int MORE = A_MORE ? S::A_DMA : S::B_DMA, LESS = S::DMA - MORE;
    auto load_both = [&](int kt, auto sac, auto sbc, auto dc) {
      constexpr int d = A_MORE ? (decltype(dc)::value + S::A_DMA) % S::DMA : decltype(dc)::value;
      if constexpr (d < S::A_DMA)
        dma_piece(kt + NSA, sac, std::integral_constant<int, d>{});
      else
        dma_piece(kt + NSB, sbc, std::integral_constant<int, d>{});
    };
    auto step = [&](int kt, auto sac, auto sbc) {
      substep(B0{}, sac, sbc, 1, B0{}, [](auto) {});
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(MORE) : "memory");
      substep(B1{}, std::integral_constant<int, (decltype(sac)::value + 1) % NSA>{}, std::integral_constant<int, (decltype(sbc)::value + 1) % NSB>{}, 0,
              DA{}, [&](auto dc) { load_both(kt, sac, sbc, dc); });
    };
    static_for<2>([&](auto sc) { static_for<S::DMA>([&](auto dc) { dma_piece(decltype(sc)::value, sc, dc); }); });
    static_for<MORE>([&](auto dc) {
      dma_piece(2, std::integral_constant<int, 2>{}, std::integral_constant<int, (A_MORE ? 0 : S::A_DMA) + decltype(dc)::value>{});
    });
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(S::DMA + MORE) : "memory");  // step 0 landed
    static_for<RD>([&](auto rc) { read_one(B0{}, B0{}, 0, 0, rc); });
    for (int kt = 0; kt < nk; kt += 6) {
      static_for<6>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        if (s == 0 || kt + s < nk) step(kt + s, std::integral_constant<int, s % NSA>{}, std::integral_constant<int, s % NSB>{});
      });
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // no LDS DMA may outlive the workgroup
  } else {
    constexpr int NS = NSA;
    using DH = std::integral_constant<int, NS == 2 ? 0 : S::DMA / 2>;  // pieces left for the next step's first half
    using DL = std::integral_constant<int, S::DMA - DH::value>;
    auto step = [&](int kt, auto slotc) {
      using Next = std::integral_constant<int, (decltype(slotc)::value + 1) % NS>;
      using Prev = std::integral_constant<int, (decltype(slotc)::value + NS - 1) % NS>;
      substep(B0{}, slotc, slotc, 1, DH{},
              [&](auto dc) { dma_piece(kt + NS - 1, Prev{}, std::integral_constant<int, DL::value + decltype(dc)::value>{}); });
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((NS - 2) * S::DMA) : "memory");
      substep(B1{}, Next{}, Next{}, 0, DL{}, [&](auto dc) { dma_piece(kt + NS, slotc, dc); });
    };
    auto fill = [&](auto sc) {
      static_for<S::DMA>([&](auto dc) {
        if constexpr (NS == 2 || decltype(sc)::value < NS - 1 || decltype(dc)::value < DL::value) dma_piece(decltype(sc)::value, sc, dc);
      });
    };
    fill(B0{});
    fill(B1{});
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(S::DMA) : "memory");  // step 0 landed
    static_for<RD>([&](auto rc) { read_one(B0{}, B0{}, 0, 0, rc); });
    static_for<NS - 2>([&](auto sc) { fill(std::integral_constant<int, decltype(sc)::value + 2>{}); });
    for (int kt = 0; kt < nk; kt += NS) {
      static_for<NS>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        if (s == 0 || kt + s < nk) step(kt + s, sc);
      });
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // no LDS DMA may outlive the workgroup
  }

  // ---- epilogue: acc[i][j][e] = product of row 16i + r16 and B tile row 16j + 4G + e of the wave's block ----
  const int mw = m0 + wm * S::WTM;
  const int nw = n0 + wn * (GATED ? S::WTN / 2 : S::WTN);
  if constexpr (SPLITK) {
    // sums of 32 bits, [split][batch][product][M][ld_part]; ld_part is a multiple of 4
    constexpr int NP = GATED ? 2 : 1;
    uint32_t* part = (uint32_t*)p.partials + ((int64_t)ks * p.batch + bz) * NP * M * p.ld_part;
    static_for<FM * FN>([&](auto xc) {
      constexpr int x = decltype(xc)::value, j = x % FN;
      const int64_t m = mw + 16 * (x / FN) + r16;
      const int n = nw + 16 * (GATED ? j / 2 : j) + 4 * G;
      if (m < M && n < N) *(u32x4*)(part + ((GATED ? (j & 1) * (int64_t)M : 0) + m) * p.ld_part + n) = __builtin_bit_cast(u32x4, acc[x / FN][j]);
    });
    return;
  }
  // Scales and bias of the tile wait in LDS: read from memory for each block they would queue behind the
  // stores of the block before.
  float* sa = (float*)smem;           // [BM] scales of a's rows
  float* sb = sa + BM;                // [2][OBN] scales of b's rows
  float* sbias = sb + 2 * OBN;        // [OBN]
  if constexpr (CODES) {
    __syncthreads();
    for (int i = tid; i < BM; i += 64 * S::NW) sa[i] = m0 + i < M ? p.a_scale[m0 + i] : 0.f;
    for (int i = tid; i < OBN; i += 64 * S::NW) {
      const bool in = n0 + i < N;
      sb[i] = in ? p.b_scale[0][n0 + i] : 0.f;
      if (GATED) sb[OBN + i] = in ? p.b_scale[1][n0 + i] : 0.f;
      if (!GATED) sbias[i] = in && p.bias != nullptr ? load_elem(p.bias, n0 + i, p.out_dtype) : 0.f;
    }
    __syncthreads();
  }
  float unit[FM];  // of the rows: read before the stores, behind which they would wait
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = mw + 16 * i + r16;
    unit[i] = m < M ? row_unit<T, MODE>(p, bz, m) : 1.f;
  }
  // four results of row block i and column block q: columns 16q + 4G .. +3 of the wave's block
  auto scaled = [&](int i, int j, int q, int half) {
    f32x4 v;
    if constexpr (CODES) {
      const RowScaled scale(sa[wm * S::WTM + 16 * i + r16]);
      const f32x4 bs = *(const f32x4*)(sb + half * OBN + (nw - n0) + 16 * q + 4 * G);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = scale((float)acc[i][j][e], bs[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * unit[i];
    }
    return v;
  };
  void* out = p.out[SUM || GATED || CODES ? 0 : bz];
  const int64_t ldo = p.ldo[SUM || GATED || CODES ? 0 : bz];
  const bool st16 = ((ldo * (int64_t)sizeof(O)) & 15) == 0 && ((uintptr_t)out & 15) == 0;
  auto finish = [&](auto actc) {
    static_for<FM>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      const int m = mw + 16 * i + r16;
      auto result = [&](auto qc) {
        constexpr int q = decltype(qc)::value;
        if constexpr (GATED) {
          const f32x4 g = scaled(i, 2 * q, q, 0), u = scaled(i, 2 * q + 1, q, 1);
          if constexpr (!CODES) {
            if (p.pre[0] != nullptr && m < M) {
              const int n = nw + 16 * q + 4 * G;
              float* pg = p.pre[0] + (int64_t)m * p.ld_pre + n;
              float* pu = p.pre[1] + (int64_t)m * p.ld_pre + n;
              if (n + 4 <= N && p.pre_vec) {
                *(f32x4*)pg = g;
                *(f32x4*)pu = u;
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (n + e < N) pg[e] = g[e], pu[e] = u[e];
              }
            }
          }
          f32x4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = act_value<decltype(actc)::value>(g[e]) * u[e];
          return y;
        } else {
          f32x4 y = scaled(i, q, q, 0);
          if constexpr (CODES) {
            const f32x4 bias = *(const f32x4*)(sbias + (nw - n0) + 16 * q + 4 * G);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += bias[e];
          }
          return y;
        }
      };
      static_for<(GATED ? FN / 2 : FN) / 2>([&](auto hc) {
        constexpr int q = 2 * decltype(hc)::value;
        const f32x4 y0 = result(std::integral_constant<int, q>{}), y1 = result(std::integral_constant<int, q + 1>{});
        if constexpr (sizeof(O) == 4) {
          static_for<2>([&](auto tc) {
            const f32x4 y = decltype(tc)::value ? y1 : y0;
            const int n = nw + 16 * (q + decltype(tc)::value) + 4 * G;
            float* dst = (float*)out + (int64_t)m * ldo + n;
            if (m < M && n + 4 <= N && st16) {
              *(f32x4*)dst = y;
            } else if (m < M) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n + e < N) dst[e] = y[e];
            }
          });
        } else {
          // one v_permlane16_swap per dword gives every lane eight consecutive columns: 16-byte stores
          uint32_t P0[2] = {pack2<O>(y0[0], y0[1]), pack2<O>(y0[2], y0[3])};
          uint32_t P1[2] = {pack2<O>(y1[0], y1[1]), pack2<O>(y1[2], y1[3])};
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const auto sw = __builtin_amdgcn_permlane16_swap(P0[w], P1[w], false, false);
            P0[w] = sw[0];
            P1[w] = sw[1];
          }
          const int n = nw + 16 * (q + (G & 1)) + 8 * (G >> 1);
          if (m < M && n < N) {
            uint16_t* dst = (uint16_t*)out + (int64_t)m * ldo + n;
            const u32x4 v = {P0[0], P0[1], P1[0], P1[1]};
            typedef u32x4 u32x4_e2 __attribute__((aligned(2)));
            if (n + 8 <= N && st16) {
              *(u32x4*)dst = v;
            } else if (n + 8 <= N) {  // rows of any pitch: one store all the same, aligned to an element
              *(u32x4_e2*)dst = v;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (n + e < N) dst[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
            }
          }
        }
      });
    });
  };
  if constexpr (GATED)
    with_act(p.act, finish);
  else
    finish(std::integral_constant<int, 0>{});
}

// 256 x 256 tiles, k of whole steps: rings of two steps of one operand and three of the other fill the LDS of a CU (160 KiB).
// The operand that more often comes from HBM, the weights (for their gradients dgate and dup), has a
// step more to arrive.  MI355X, rings of two steps -> this: gated bf16 4096 x 4096, two of 14336, 707 -> 650 us, codes 4096 x 14336
// x 4096 177 -> 163, dx 672 -> 650, dw 696 -> 681.  (128 x 128 tiles gain 0 to 3 % where they are chosen, for three
// times the code; with the checks of a partial step dx would spill registers.)
// Tiles: 256 x 256 with 8 waves, one workgroup per CU; 128 x 128 with 4 waves, two per CU, or one with
// a ring of four steps where no CU gets a second (see the plan); and, along k, 256 x 128 with 8 waves and a ring
// of three steps, for some hundred rows whose weights come from HBM: the time is that of loads on their way (x[256,
// 4096], two weights of 14336 rows, bf16: 256 x 256 101 us, 128 x 128 85, 256 x 128 with a ring of two 84, of three 68).
template <typename T, typename O, int MODE, bool AKM, bool BKN, bool KCHECK>
hipError_t launch_projection_tile_k(const ProjParams& p, int bm, int bn, bool deep, dim3 grid, hipStream_t s) {
  constexpr int A2 = AKM && !KCHECK ? 3 : 2, B2 = AKM || KCHECK ? 2 : 3;
  if constexpr (!AKM && !BKN) {
    if (bn == 128 && bm == 256)
      return launch_kernel((projection_tile_kernel<T, O, MODE, AKM, BKN, 256, 128, 4, 2, 1, 3, 3, KCHECK, false>), grid, dim3(512), 0, s, p);
  }
  if (bm == 256)
    return launch_kernel((projection_tile_kernel<T, O, MODE, AKM, BKN, 256, 256, 4, 2, 1, A2, B2, KCHECK, false>), grid, dim3(512), 0, s, p);
  if (p.splits > 1) {
    if (deep)
      return launch_kernel((projection_tile_kernel<T, O, MODE, AKM, BKN, 128, 128, 2, 2, 1, 4, 4, KCHECK, true>), grid, dim3(256), 0, s, p);
    return launch_kernel((projection_tile_kernel<T, O, MODE, AKM, BKN, 128, 128, 2, 2, 2, 2, 2, KCHECK, true>), grid, dim3(256), 0, s, p);
  }
  if (deep)
    return launch_kernel((projection_tile_kernel<T, O, MODE, AKM, BKN, 128, 128, 2, 2, 1, 4, 4, KCHECK, false>), grid, dim3(256), 0, s, p);
  return launch_kernel((projection_tile_kernel<T, O, MODE, AKM, BKN, 128, 128, 2, 2, 2, 2, 2, KCHECK, false>), grid, dim3(256), 0, s, p);
}

template <typename T, typename O, int MODE, bool AKM, bool BKN>
hipError_t launch_projection_tile(const ProjParams& p, int bm, int bn, bool deep, hipStream_t s) {
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)(p.batch * p.splits));
  constexpr int BK = 128 / sizeof(T);
  if (p.K % BK != 0) return launch_projection_tile_k<T, O, MODE, AKM, BKN, true>(p, bm, bn, deep, grid, s);
  return launch_projection_tile_k<T, O, MODE, AKM, BKN, false>(p, bm, bn, deep, grid, s);
}

}  // namespace cmpext3
