// Attention over many query rows (gfx950): O = softmax(scale Q K^T) V in one pass over the
// keys with the running maximum and sum of the softmax.
//
// Rows: a workgroup takes NW x 32 rows of one sequence and one kv head, a row being one
// query of one head of the group (row r: query r / group, head r % group), so that grouped
// heads share each step's keys and values and short sequences fill their tiles.  A wave owns
// 32 rows.
//
// Products (32x32x16, fp32 sums) run transposed: S^T = K Q^T gives lane l the scores of row
// l % 32 only (keys 8 (r / 4) + 4 (l / 32) + r % 4 of a block of 32), so the maximum, sum and
// scale of a row are one register of a lane, joined over the two half-waves by one exchange;
// and the weights are at once the second operand of O^T = V^T P^T, if the k slots of that
// product take the keys in the order the lane has them: the transposing LDS reads of V then
// fetch rows 16 g + 4 (l / 32) and + 8 instead of 8 consecutive ones.  No weight crosses lanes.
//
// The maximum a row subtracts is only raised when a score exceeds it by more than 2^8
// (kLazy): the sums stay far from overflow and the accumulators are rarely rescaled.
//
// Keys and values of a step (64 keys) lie in LDS as rows of HD 16-bit elements in one of two
// slots, K with its 16-byte chunks and V with its 64-byte segments permuted by the row so
// that the reads of both products hit all banks.  Packed ones come by LDS DMA, which zero
// fills what lies past the sequence or the head; pages are read into registers (any page
// size, 8-bit codes converted on the way) and stored.  One barrier a step: the next step's
// loads start behind it, into the slot the step before has read.
#pragma once

#include "attention_common.h"

namespace cmpext3 {

constexpr float kLazy = 8.0f;  // in powers of two

template <int HD, int NW, bool PAGED>
struct TileShape {
  static constexpr int BM = 32 * NW;
  static constexpr int ROW = HD * 2;              // bytes of a key's row in LDS
  static constexpr int BYTES = kTileKeys * ROW;   // K or V of a step
  static constexpr int SLOT = 2 * BYTES;
  static constexpr int SCALES = 2 * kTileKeys * 4;  // 8-bit: the step's scales of K and V
  static constexpr int LDS = 2 * SLOT + (PAGED ? 2 * SCALES : 0);
  static constexpr int DMA = BYTES / 1024 / NW;  // 1 KB LDS-DMA loads per wave of K, and of V
  static_assert(BYTES % (1024 * NW) == 0, "whole DMA loads per wave");
};

// Byte offset in a K slot of the 16-byte chunk `chunk` of row `row`: 16 rows at one chunk
// cover the 16 chunk places of 256 bytes.
template <int HD>
__device__ __forceinline__ int k_place(int row, int chunk) {
  if constexpr (HD == 64) {
    const int p = row >> 1;
    return p * 256 + ((row & 1) << 7) + (((chunk ^ p) & 7) << 4);
  } else {
    return row * HD * 2 + (((chunk & ~15) | ((chunk ^ row) & 15)) << 4);
  }
}
// The same for V, 64-byte segments (32 columns): four consecutive rows at one segment cover
// 256 bytes.
template <int HD>
__device__ __forceinline__ int v_place(int row, int byte_col) {
  const int x = HD == 64 ? (row >> 1) & 1 : row & 3;
  return row * HD * 2 + (((byte_col >> 6) ^ x) << 6) + (byte_col & 63);
}

template <typename T, int HD, int KIND, int NW>
__global__ void __launch_bounds__(64 * NW, HD <= 128 ? 8 / NW : 1) attention_tile_kernel(const AttnParams p) {
  constexpr bool kPaged = KIND != kKvPacked, k8 = KIND == kKvPaged8;
  using S = TileShape<HD, NW, kPaged>;
  constexpr int KK = HD / 16, DB = HD / 32;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[S::LDS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;

  // heads fastest: the workgroups of one kv head meet in the L2 of few XCDs
  const int kvh = blockIdx.x % p.kv_heads;
  Seq sq = seq_of_slot(p, blockIdx.x / p.kv_heads, S::BM);
  if (sq.b < 0) return;
  const int split = blockIdx.y;
  const int shift = sq.len_k - sq.len_q;  // causal: query i sees keys up to i + shift
  const int row0 = sq.tile * S::BM, rows = sq.len_q * p.group;
  // keys any row of the tile sees
  const int last_q = min(row0 + S::BM, rows) - 1;
  int end = sq.len_k;
  if (p.causal) end = min(end, last_q / p.group + shift + 1);
  const int begin = split * p.split_keys;
  end = min(end, begin + p.split_keys);
  if (p.splits > 1 && begin >= sq.len_k && split > 0) return;  // this split has no keys: the join knows

  // ---- this lane's row ----
  const int row = row0 + wave * 32 + col;
  const bool live = row < rows;
  const int tok = min(row, rows - 1) / p.group;
  const int head = kvh * p.group + (min(row, rows - 1) - tok * p.group);
  const int last = min(sq.len_k, end) - 1;  // keys past `end` are another split's
  const int limit = p.causal ? min(tok + shift, last) : last;  // its last key
  const int wtok0 = min(row0 + wave * 32, rows - 1) / p.group;
  const int wtok1 = min(row0 + wave * 32 + 31, rows - 1) / p.group;
  // keys that all rows of the wave see, and that any of them sees
  const int wave_all = __builtin_amdgcn_readfirstlane(p.causal ? min(wtok0 + shift, last) : last);
  const int wave_any = __builtin_amdgcn_readfirstlane(
      row0 + wave * 32 < rows ? (p.causal ? min(wtok1 + shift, last) : last) : -1);

  u32x4 q[KK];
  {
    const T* qp = (const T*)p.q + sq.b * p.q_batch + (int64_t)(sq.q0 + tok) * p.q_token + (int64_t)head * p.q_head;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = 16 * kk + 8 * half;
      q[kk] = live && d < p.dim ? *(const u32x4*)(qp + d) : u32x4{0, 0, 0, 0};
    }
  }

  // ---- loads of a step ----
  const int32_t* table = kPaged ? p.kv.table + sq.b * p.kv.table_row : nullptr;
  const T* kbase = nullptr;
  const T* vbase = nullptr;
  uint32_t k_off[kPaged ? 1 : S::DMA], v_off[kPaged ? 1 : S::DMA];
  int k_row[kPaged ? 1 : S::DMA], v_row[kPaged ? 1 : S::DMA];
  if constexpr (!kPaged) {
    kbase = (const T*)p.kv.k + sq.b * p.kv.k_page + (int64_t)sq.k0 * p.kv.k_token + (int64_t)kvh * p.kv.k_head;
    vbase = (const T*)p.kv.v + sq.b * p.kv.v_page + (int64_t)sq.k0 * p.kv.v_token + (int64_t)kvh * p.kv.v_head;
#pragma unroll
    for (int i = 0; i < S::DMA; ++i) {
      const int pos = (wave * S::DMA + i) * 1024 + 16 * lane;
      int c;
      if constexpr (HD == 64) {
        const int pr = pos >> 8, c16 = (pos & 255) >> 4;
        k_row[i] = 2 * pr + (c16 >> 3);
        c = (c16 ^ pr) & 7;
      } else {
        k_row[i] = pos / S::ROW;
        const int c16 = (pos % S::ROW) >> 4;
        c = (c16 & ~15) | ((c16 ^ k_row[i]) & 15);
      }
      k_off[i] = 8 * c < p.dim ? (uint32_t)(k_row[i] * (int)p.kv.k_token + 8 * c) * 2u : kBufOOB;
      v_row[i] = pos / S::ROW;
      const int x = HD == 64 ? (v_row[i] >> 1) & 1 : v_row[i] & 3;
      const int bc = ((((pos % S::ROW) >> 6) ^ x) << 6) + (pos & 63);
      v_off[i] = bc < 2 * p.dim ? (uint32_t)(v_row[i] * (int)p.kv.v_token * 2 + bc) : kBufOOB;
    }
  }
  // paged: 16-byte pieces of a step, in the order of the cache
  constexpr int EPP = k8 ? 16 : 8;                                // elements of a piece
  constexpr int PIECES = kTileKeys * HD / EPP / (64 * NW);        // per thread, of K and of V
  constexpr int PPR = HD / EPP;                                   // pieces of a row
  u32x4 kreg[kPaged ? PIECES : 1], vreg[kPaged ? PIECES : 1];
  float sreg = 0.f;
  auto load = [&](int key0, int slot) {
    if constexpr (!kPaged) {
      const int left = sq.len_k - key0;
      const i32x4 kr = make_rsrc_sgpr(kbase + (int64_t)key0 * p.kv.k_token);
      const i32x4 vr = make_rsrc_sgpr(vbase + (int64_t)key0 * p.kv.v_token);
      const uint32_t dst = lds_addr(smem) + (uint32_t)(slot * S::SLOT + wave * S::DMA * 1024);
      static_for<S::DMA>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        dma_load16_m0(kr, k_row[i] < left ? k_off[i] : kBufOOB, 0, dst,
                      std::integral_constant<uint32_t, i * 1024>{});
      });
      static_for<S::DMA>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        dma_load16_m0(vr, v_row[i] < left ? v_off[i] : kBufOOB, 0, dst,
                      std::integral_constant<uint32_t, S::BYTES + i * 1024>{});
      });
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int n = i * 64 * NW + tid, r = n / PPR, d = (n % PPR) * EPP;
        const int key = key0 + r;
        kreg[i] = vreg[i] = u32x4{0, 0, 0, 0};
        if (key < sq.len_k && d < p.dim) {
          int place;
          const int page = page_of(p.kv, table, key, place);
          if (page >= 0) {
            const int64_t ko = page * p.kv.k_page + place * p.kv.k_token + kvh * p.kv.k_head + d;
            const int64_t vo = page * p.kv.v_page + place * p.kv.v_token + kvh * p.kv.v_head + d;
            if (k8 && d + 8 >= p.dim) {  // a row of an odd number of 8-byte pieces ends here
              const u32x2 a = *(const u32x2*)((const uint8_t*)p.kv.k + ko), b = *(const u32x2*)((const uint8_t*)p.kv.v + vo);
              kreg[i].x = a.x, kreg[i].y = a.y, vreg[i].x = b.x, vreg[i].y = b.y;
            } else {
              constexpr int es = k8 ? 1 : 2;
              kreg[i] = *(const u32x4_a8*)((const uint8_t*)p.kv.k + ko * es);
              vreg[i] = *(const u32x4_a8*)((const uint8_t*)p.kv.v + vo * es);
            }
          }
        }
      }
      if constexpr (k8) {
        if (tid < 2 * kTileKeys) {
          const int key = key0 + (tid & (kTileKeys - 1));
          sreg = 0.f;
          if (key < sq.len_k) {
            int place;
            const int page = page_of(p.kv, table, key, place);
            if (page >= 0)
              sreg = tid < kTileKeys
                         ? p.kv.k_scale[page * p.kv.ks_page + place * p.kv.ks_token + kvh * p.kv.ks_head] * p.scale_log2
                         : p.kv.v_scale[page * p.kv.vs_page + place * p.kv.vs_token + kvh * p.kv.vs_head];
          }
        }
      }
    }
  };
  auto store = [&](int slot) {
    if constexpr (kPaged) {
      unsigned char* ks = smem + slot * S::SLOT;
      unsigned char* vs = ks + S::BYTES;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int n = i * 64 * NW + tid, r = n / PPR, c = (n % PPR) * (EPP / 8);
        if constexpr (k8) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const u32x2 a = e4m3x4<T>(kreg[i][2 * h]), b = e4m3x4<T>(kreg[i][2 * h + 1]);
            *(u32x4*)(ks + k_place<HD>(r, c + h)) = u32x4{a.x, a.y, b.x, b.y};
            const u32x2 e = e4m3x4<T>(vreg[i][2 * h]), f = e4m3x4<T>(vreg[i][2 * h + 1]);
            *(u32x4*)(vs + v_place<HD>(r, 16 * (c + h))) = u32x4{e.x, e.y, f.x, f.y};
          }
        } else {
          *(u32x4*)(ks + k_place<HD>(r, c)) = kreg[i];
          *(u32x4*)(vs + v_place<HD>(r, 16 * c)) = vreg[i];
        }
      }
      if constexpr (k8)
        if (tid < 2 * kTileKeys) *(float*)(smem + 2 * S::SLOT + slot * S::SCALES + 4 * tid) = sreg;
    }
  };

  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x16{0};
  float m_ref = -INFINITY;  // what the row's weights are relative to (in units of `unit`)
  float sum = 0.f;          // of this lane's keys only
  const float unit = k8 ? 1.f : p.scale_log2;  // scores times this are powers of two

  // LDS offsets of this lane's fragments: K's row `col` at chunk 2 kk + half (the second block
  // of 32 keys lies a fixed distance on), V's transposing reads: row 4 half + r16 / 4, columns
  // 32 d + 16 (G % 2) + 4 (r16 % 4) (further rows, multiples of 8, keep the permutation)
  int k_at[KK], v_at[DB];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) k_at[kk] = k_place<HD>(col, 2 * kk + half);
#pragma unroll
  for (int d = 0; d < DB; ++d)
    v_at[d] = S::BYTES + v_place<HD>(4 * half + ((lane & 15) >> 2), 2 * (32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)));

  auto v_frag = [&](const unsigned char* slot, int g, int d) {
    const u32x2 lo = lds_read_tr(slot + v_at[d] + 16 * g * S::ROW);
    const u32x2 hi = lds_read_tr(slot + v_at[d] + (16 * g + 8) * S::ROW);
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };
  // masked: some row of the wave does not see all 64 keys
  auto compute = [&](int key0, int slot, bool masked) {
    const unsigned char* ks = smem + slot * S::SLOT;
    f32x16 s[2] = {f32x16{0}, f32x16{0}};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const u32x4 k = *(const u32x4*)(ks + k_at[kk] + b * 32 * S::ROW);
        s[b] = Mfma32<T>::mma(k, q[kk], s[b]);
      }
      if (kk % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // no more fragments at once than four
    }
    const float* sc = (const float*)(smem + 2 * S::SLOT + slot * S::SCALES);
    if constexpr (k8) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] *= sc[32 * b + 8 * (r / 4) + 4 * half + r % 4];
    }
    if (masked) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[b][r] = key0 + 32 * b + 8 * (r / 4) + 4 * half + r % 4 <= limit ? s[b][r] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int r = 1; r < 32; ++r) mx = fmaxf(mx, s[r / 16][r % 16]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__builtin_amdgcn_ballot_w64((mx - m_ref) * unit > kLazy)) {  // -inf - -inf is no reason
      const float m_new = fmaxf(m_ref, mx);
      const float alpha = m_new == m_ref ? 1.f : exp2_hw((m_ref - m_new) * unit);
      m_ref = m_new;
      sum *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
    const float base = m_ref == -INFINITY ? 0.f : m_ref * unit;
    u32x4 pw[4];  // weights of 16 keys each
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        float w0, w1;
        if constexpr (k8) {
          w0 = exp2_hw(s[b][r] - base);
          w1 = exp2_hw(s[b][r + 1] - base);
        } else {
          w0 = exp2_hw(__builtin_fmaf(s[b][r], unit, -base));
          w1 = exp2_hw(__builtin_fmaf(s[b][r + 1], unit, -base));
        }
        sum += w0 + w1;
        if constexpr (k8) {
          const int key = 32 * b + 8 * (r / 4) + 4 * half + r % 4;
          w0 *= sc[kTileKeys + key];
          w1 *= sc[kTileKeys + key + 1];
        }
        pw[2 * b + r / 8][(r % 8) / 2] = pack2<T>(w0, w1);
      }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] = Mfma32<T>::mma(v_frag(ks, g, d), pw[g], o[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // keys that all rows of the workgroup see
  const int tile_all = p.causal ? min(row0 / p.group + shift, last) : last;
  bool spoilt = false;
  if (begin < end) {
    load(begin, 0);
    store(0);
    int slot = 0;
    for (int key0 = begin; key0 < end; key0 += kTileKeys) {
      ring_fence<0>();  // this step's keys and values are in LDS, and the other slot is read
      if (key0 + kTileKeys < end) load(key0 + kTileKeys, slot ^ 1);
      if (key0 + kTileKeys - 1 > tile_all) {
        unsigned char* vs = smem + slot * S::SLOT + S::BYTES;
        if (any_not_finite<T>(vs, S::BYTES)) {  // all waves find the same
          spoilt = true;
          __syncthreads();
          for (int i = 16 * tid; i < S::BYTES; i += 16 * 64 * NW) *(u32x4*)(vs + i) = finite_only<T>(*(const u32x4*)(vs + i));
          __syncthreads();
        }
      }
      if (key0 <= wave_any) compute(key0, slot, key0 + kTileKeys - 1 > wave_all);
      if (key0 + kTileKeys < end) store(slot ^ 1);
      slot ^= 1;
    }
  }

  if (spoilt) {  // add what was made zero (see any_not_finite)
    for (int key0 = begin; key0 < end; key0 += kTileKeys) {
      if (key0 + kTileKeys - 1 <= tile_all) continue;
      ring_fence<0>();  // slot 0 is read
      load(key0, 0);
      store(0);
      ring_fence<0>();
      for (int kind = 0; kind < 3; ++kind)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          f32x16 hit = f32x16{0};
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int key = key0 + 16 * g + 4 * half;
            const u32x4 seen = {ones_up_to<T>(key, limit), ones_up_to<T>(key + 2, limit), ones_up_to<T>(key + 8, limit),
                                ones_up_to<T>(key + 10, limit)};
            hit = Mfma32<T>::mma(kind_ones<T>(v_frag(smem, g, d), kind), seen, hit);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] += hit[r] > 0.f ? kind_value(kind) : 0.f;
        }
    }
  }

  // ---- out: lane has row `row`, elements 32 d + 8 (r / 4) + 4 half + r % 4 ----
  sum += __shfl_xor(sum, 32);
  if (!live) return;
  if (p.splits > 1) {
    const int64_t at = (int64_t)split * p.rows + ((int64_t)sq.b * (p.starts_q ? 0 : p.len_q) + sq.q0 + tok) * p.heads + head;
    float* po = p.part_o + at * p.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int e = 32 * d + 8 * (r / 4) + 4 * half;
        if (e < p.dim) *(f32x4*)(po + e) = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
      }
    if (half == 0) {
      p.part_ml[2 * at] = m_ref * unit;
      p.part_ml[2 * at + 1] = sum;
    }
    return;
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  T* op = (T*)p.out + sq.b * p.out_batch + (int64_t)(sq.q0 + tok) * p.out_token + (int64_t)head * p.out_head;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int e = 32 * d + 8 * (r / 4) + 4 * half;
      if (e < p.dim)
        *(u32x2*)(op + e) = u32x2{pack2<T>(o[d][r] * inv, o[d][r + 1] * inv), pack2<T>(o[d][r + 2] * inv, o[d][r + 3] * inv)};
    }
}

template <typename T, int HD, int KIND>
hipError_t launch_tile_kind(const AttnParams& p, dim3 grid, hipStream_t s) {
  return launch_kernel(attention_tile_kernel<T, HD, KIND, 4>, grid, dim3(256), 0, s, p);
}
template <typename T, int KIND>
hipError_t launch_tile_hd(int hd, const AttnParams& p, dim3 grid, hipStream_t s) {
  if (hd == 64) return launch_tile_kind<T, 64, KIND>(p, grid, s);
  if (hd == 128) return launch_tile_kind<T, 128, KIND>(p, grid, s);
  return launch_tile_kind<T, 256, KIND>(p, grid, s);
}

}  // namespace cmpext3
