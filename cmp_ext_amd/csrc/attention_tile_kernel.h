// Attention over many query rows (gfx950): O = softmax(scale Q K^T) V in one pass over the
// keys with the running maximum and sum of the softmax.
//
// Rows: a workgroup of four waves takes 128 rows of one sequence and one kv head, a row being one
// query of one head of the group (row r: query r / group, head r % group), so that grouped heads
// share each step's keys and values and short sequences fill their tiles.  A wave owns 32 rows.
// (8192 tokens, 32 heads of 128 and 8 of keys, bf16, on MI355X: 512 us, 503 to 520 on different boxes,
// 1074 TFLOP/s of the products that are not masked.  When four waves of 32 rows took 529, eight over 256 rows,
// whose barriers bind all waves of a CU together, took 548, and four of 64 rows with a SIMD to themselves 643.)
//
// Keys: where there are fewer tiles than CUs, a workgroup has two such groups of four waves (KS = 2),
// one for the even steps and one for the odd ones, each with its own LDS, joined in LDS at the end:
// two waves on every SIMD as with two workgroups, and half as many steps.  Beyond that the keys
// are split over workgroups (attention_join.h).
//
// Products (32x32x16, fp32 sums) run transposed: S^T = K Q^T gives lane l the scores of row
// l % 32 only (keys 8 (r / 4) + 4 (l / 32) + r % 4 of a block of 32), so the maximum, sum and
// scale of a row are one register of a lane, joined over the two half-waves by one exchange;
// and the weights are at once the second operand of O^T = V^T P^T, if the k slots of that
// product take the keys in the order the lane has them: the transposing LDS reads of V then
// fetch rows 16 g + 4 (l / 32) and + 8 instead of 8 consecutive ones.  No weight crosses lanes.
//
// The maximum a row subtracts is only raised when a score exceeds it by more than 2^8 (2^4 in fp16,
// where the weights begin at 2^10: see kHalf): the sums stay far from overflow and the accumulators are
// rarely rescaled.
//
// Pipeline: step j (64 keys) has two phases, each a sequence of slots of one matrix product with
// a share of the vector work, kept in that order: the scores of step j + 1 beside the first
// weights of step j, then the weighted values of step j beside its other weights and the maximum
// of step j + 1.  The vector work (per score: scale, exponential at half the rate, sum, half a
// conversion, half a maximum) is over half as long as the products.  On that prompt the matrix cores
// are busy 56 % of the cycles and the vector units 49 %, a wave waits for LDS or its barrier 23 % of its
// time, and power bounds it as well: 1339 W of the board's 1400, at 1.79 GHz (2.4 under the other kernels
// here).  More fragments on their way, or other shares of the vector work in the two phases, changed nothing.
//
// The weights are rounded once to 16 bits for the second product, their sum is of the unrounded
// ones: the result is off by its own rounding and by one of the same size more (in fp16 for weights down to
// 2^-24 of the row's largest; over codes, down to 2^-20 of the largest times the largest scale among the 64 keys
// of a step; below that a weight is off by up to 2^-35, or 2^-31, of that).
//
// Keys and values of a step lie in LDS as rows of HD 16-bit elements in two slots each, K
// with its 16-byte chunks and V with its 64-byte segments permuted by the row so that the reads
// of both products hit all banks.  16-bit ones come by LDS DMA, packed through a descriptor that
// zero fills what lies past the sequence or the head, pages (of any size) from each lane's own
// address or a piece of zeros (through registers instead: 6 chunks of up to 512 over up to 4000
// keys, heads 16 / 4, 75.6 us for 67.0, one of 1024 over 4096, heads 32 / 8, 95.7 for 89.2).  8-bit codes are
// converted on the way, in registers (one set of them, for K in the first phase and V in the
// second: with two, 93 spills made chunks 206 us instead of 141; 126 with what followed, 4 of up to 512
// over up to 8100 keys, heads 32 / 8).  The rows' addresses in the pages are
// shared through LDS, their page numbers fetched steps ahead.  One barrier a step: K of step j + 2 and V of step j + 1 start to load
// behind it, into the slots that the step before has read; they land well within a step.
#pragma once

#include "attention_join.h"

namespace cmpext3 {

constexpr int kTileWaves = 4;

constexpr int kSlots = 2;  // of K and of V

template <int HD, bool PAGED>
struct TileShape {
  static constexpr int ROW = HD * 2;             // bytes of a key's row in LDS
  static constexpr int BYTES = kTileKeys * ROW;  // K or V of a step
  static constexpr int V0 = kSlots * BYTES;          // K's slots, then V's
  static constexpr int ROWS_AT = 2 * kSlots * BYTES;  // paged: byte offsets of the rows of K and V, two steps'
  static constexpr int SCALES = ROWS_AT + 2 * 2 * kTileKeys * 8;  // 8 bits: scales of K and V, four steps'
  static constexpr int UNITS = SCALES + 4 * 2 * kTileKeys * 4;    // and the unit of V's, four steps'
  static constexpr int LDS = PAGED ? UNITS + 4 * 4 : ROWS_AT;
  static constexpr int DMA = BYTES / 1024 / kTileWaves;  // 1 KB LDS-DMA loads per wave of K, and of V
  static_assert(BYTES % (1024 * kTileWaves) == 0, "whole DMA loads per wave");
  static_assert(LDS <= 160 * 1024 && LDS >= kJoinBytes, "LDS budget");
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

// What LDS-DMA reads for rows that are not there.
static __device__ const uint32_t zero_piece[4] __attribute__((aligned(16))) = {0, 0, 0, 0};

// Two waves share a SIMD's registers (packed heads up to 64: three; over 128: one has them all).
template <typename T, int HD, int KIND, int KS>
__global__ void __launch_bounds__(64 * kTileWaves * KS, HD == 256 ? 1 : HD == 64 && KIND == kKvPacked && KS == 1 ? 3 : 2) attention_tile_kernel(const AttnParams p) {
  constexpr bool kPaged = KIND != kKvPacked, k8 = KIND == kKvPaged8;
  using S = TileShape<HD, kPaged>;
  constexpr int KK = HD / 16, DB = HD / 32, NW = kTileWaves, BM = 32 * NW;
  __shared__ __attribute__((aligned(1024))) unsigned char all_smem[S::LDS * KS];
  __shared__ int any_spoilt;

  const int tid = threadIdx.x & (64 * NW - 1), lane = tid & 63;  // of a group of four waves
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part_k = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / (64 * NW));  // which group
  unsigned char* smem = all_smem + part_k * S::LDS;
  const int half = lane >> 5, col = lane & 31;

  // heads fastest: the workgroups of one kv head meet in the L2 of few XCDs
  const int kvh = blockIdx.x % p.kv_heads;
  const Seq sq = seq_of_slot<kPaged>(p, blockIdx.x / p.kv_heads, BM);
  if (sq.b < 0) return;
  const int split = blockIdx.y;
  const int shift = sq.len_k - sq.len_q;  // causal: query i sees keys up to i + shift
  const int row0 = sq.tile * BM, rows = sq.len_q * p.group;
  int end = keys_end(p, sq, min(row0 + BM, rows) - 1);  // of the keys any row of the tile sees
  const int splits = splits_of(p, sq, end);
  if (split >= splits) return;
  // what only the end of the kernel needs waits in LDS: the loop has no register to spare
  __shared__ Seq kept_seq;
  __shared__ int kept_kvh, kept_row0, kept_splits;
  if (threadIdx.x == 0) {
    kept_seq = sq;
    kept_kvh = kvh;
    kept_row0 = row0;
    kept_splits = splits;
  }
  const int begin = split * sq.split_keys;
  end = min(end, begin + sq.split_keys);
  // steps of this group, and of the group that has most: step j starts at key key_of(j)
  const int all_steps = end > begin ? (end - begin + kTileKeys - 1) / kTileKeys : 0;
  const int steps = (all_steps - part_k + KS - 1) / KS, turns = (all_steps + KS - 1) / KS;
  auto key_of = [&](int j) { return begin + (j * KS + part_k) * kTileKeys; };

  // ---- this lane's row ----
  const int last = min(sq.len_k, end) - 1;  // keys past `end` are another split's
  const int wrow0 = row0 + wave * 32, row = wrow0 + col;
  const int tok = min(row, rows - 1) / p.group, head = kvh * p.group + min(row, rows - 1) - tok * p.group;
  const int limit = p.causal ? min(tok + shift, last) : last;  // the last key it sees
  u32x4 q[KK];
  {
    const T* qp = (const T*)p.q + sq.b * p.q_batch + (int64_t)(sq.q0 + tok) * p.q_token + (int64_t)head * p.q_head;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = 16 * kk + 8 * half;
      q[kk] = row < rows && d < p.dim ? *(const u32x4*)(qp + d) : u32x4{0, 0, 0, 0};
    }
  }
  // keys that all rows of the wave see, and that any of them sees; that all rows of the tile see
  const int wave_all = __builtin_amdgcn_readfirstlane(p.causal ? min(min(wrow0, rows - 1) / p.group + shift, last) : last);
  const int wave_any = __builtin_amdgcn_readfirstlane(
      wrow0 < rows ? (p.causal ? min((min(wrow0 + 32, rows) - 1) / p.group + shift, last) : last) : -1);
  const int tile_all = p.causal ? min(row0 / p.group + shift, last) : last;

  // ---- loads: K or V of a step into a slot ----
  // 16 bits: LDS-DMA loads i of this wave; where lane's 16 bytes of load i come from (pages: in a row)
  const T* kbase = nullptr;
  const T* vbase = nullptr;
  uint32_t k_off[S::DMA], v_off[S::DMA];
  constexpr int ROWS1K = 1024 / S::ROW;  // rows of a DMA load
  const int dma_row = wave * S::DMA * ROWS1K + 16 * lane / S::ROW;
  if constexpr (!k8) {
    kbase = (const T*)p.kv.k + sq.b * p.kv.k_page + (int64_t)sq.k0 * p.kv.k_token + (int64_t)kvh * p.kv.k_head;
    vbase = (const T*)p.kv.v + sq.b * p.kv.v_page + (int64_t)sq.k0 * p.kv.v_token + (int64_t)kvh * p.kv.v_head;
#pragma unroll
    for (int i = 0; i < S::DMA; ++i) {
      const int row = dma_row + i * ROWS1K, at = 16 * lane % S::ROW;  // bytes into the row's place
      int c;
      if constexpr (HD == 64)
        c = ((at >> 4) ^ (row >> 1)) & 7;
      else
        c = ((at >> 4) & ~15) | (((at >> 4) ^ row) & 15);
      k_off[i] = 8 * c < p.dim ? (uint32_t)((kPaged ? 0 : row * (int)p.kv.k_token) + 8 * c) * 2u : kBufOOB;
      const int x = HD == 64 ? (row >> 1) & 1 : row & 3;
      const int bc = (((at >> 6) ^ x) << 6) + (at & 63);
      v_off[i] = bc < 2 * p.dim ? (uint32_t)((kPaged ? 0 : row * (int)p.kv.v_token * 2) + bc) : kBufOOB;
    }
  }
  const uint32_t lds0 = lds_addr(smem) + (uint32_t)(wave * S::DMA * 1024);
  // K or V of the step from key0 into a slot, zeros past the sequence and of steps past the last
  auto dma = [&](bool value, int step, int slot) {
    const int key0 = key_of(step);
    const i32x4 r = make_rsrc_sgpr(value ? vbase + (int64_t)key0 * p.kv.v_token : kbase + (int64_t)key0 * p.kv.k_token);
    const uint32_t dst = lds0 + (uint32_t)((value ? S::V0 : 0) + slot * S::BYTES);
    const int left = step < steps ? sq.len_k - key0 : 0;
    if (left >= kTileKeys) {
      static_for<S::DMA>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        dma_load16_m0(r, value ? v_off[i] : k_off[i], 0, dst, std::integral_constant<uint32_t, i * 1024>{});
      });
    } else {
      static_for<S::DMA>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        dma_load16_m0(r, dma_row + i * ROWS1K < left ? (value ? v_off[i] : k_off[i]) : kBufOOB, 0, dst,
                      std::integral_constant<uint32_t, i * 1024>{});
      });
    }
  };
  // paged: thread t < 64 looks after row t of a step of K, thread 64 + t after one of V: finds its
  // page, its byte offset in the cache (rows_at[step % 2][t], -1: zeros) and its scale
  constexpr int EPP = 16, ES = k8 ? 1 : 2;                  // 8 bits: elements of a 16-byte piece; bytes of an element
  constexpr int PIECES = kTileKeys * HD / EPP / (64 * NW);  // pieces a thread loads of K, and of V
  constexpr int PPR = HD / EPP;                             // pieces of a row
  int64_t* rows_at = (int64_t*)(smem + S::ROWS_AT);
  float* scales = (float*)(smem + S::SCALES);  // [step % 4][K, V][64]
  // fp16: V's scales of a step are held in a power of two of their own size, 2^(unit - 127), and so are the
  // sums: weights that carry them stay where fp16 has its bits (see kHalf) whatever the values' size.
  // The unit is raised to the largest of a step, and lowered to it if that is over 2^4 smaller.  (4 of up to
  // 512 over up to 8100 keys, heads 32 / 8 of 128: 130 us for 127 without, of 64: 104 for 99; found by the wave that
  // stores the scales, which has most to do, 134 for heads of 128.)
  constexpr bool UNITS = k8 && kHalf<T>;
  int* units = (int*)(smem + S::UNITS);  // [step % 4]
  int unit_found = 127, most_found = 1;  // the wave that finds it: of the last step, the largest of all
  const int32_t* table = kPaged ? p.kv.table + sq.b * p.kv.table_row : nullptr;
  const bool value_row = wave > 0;  // of the first two waves, which find the rows
  u32x4 reg[PIECES];  // 8 bits: of K in a step's first phase, of V in its second
  float sreg = 0.f;
  auto page_number = [&](int key) -> int {  // of this thread's row
    if (wave > 1 || key >= sq.len_k) return -1;
    return table[p.kv.page_shift >= 0 ? key >> p.kv.page_shift : key / p.kv.page_size];
  };
  auto place_row = [&](int at, int key, int page) {
    if (wave > 1) return;
    const int place = p.kv.page_shift >= 0 ? key & (p.kv.page_size - 1) : key % p.kv.page_size;
    const bool there = (unsigned)page < (unsigned)p.kv.pages;
    const int64_t o = value_row ? page * p.kv.v_page + place * p.kv.v_token + kvh * p.kv.v_head
                                : page * p.kv.k_page + place * p.kv.k_token + kvh * p.kv.k_head;
    rows_at[at * 2 * kTileKeys + tid] = there ? o * ES : -1;
    if constexpr (k8) {
      sreg = 0.f;
      if (there)
        sreg = value_row ? p.kv.v_scale[page * p.kv.vs_page + place * p.kv.vs_token + kvh * p.kv.vs_head]
                         : p.kv.k_scale[page * p.kv.ks_page + place * p.kv.ks_token + kvh * p.kv.ks_head];
    }
  };
  auto store_scale = [&](int step_k, int step_v) {
    if (k8 && wave < 2) scales[((value_row ? step_v : step_k) & 3) * 2 * kTileKeys + tid] = sreg;
  };
  auto value_scales = [&](int step) { return scales + (step & 3) * 2 * kTileKeys + kTileKeys; };
  auto find_unit = [&](int step) {  // the last wave, which finds no rows, behind a barrier after the scales were stored
    if constexpr (UNITS) {
      if (wave != NW - 1) return;
      float* mine = value_scales(step) + lane;
      const int bits = __float_as_int(fabsf(*mine)), e = bits < 0x7F800000 ? bits >> 23 : 0;
      if (__builtin_amdgcn_ballot_w64(e > unit_found) != 0 || __builtin_amdgcn_ballot_w64(e >= unit_found - 4) == 0) {
        const int most = largest(e);  // 0: only zeros, nothing to go by
        most_found = max(most_found, most);
        if (most > 0) unit_found = max(most, most_found - 60);  // not so far below that sums of the largest leave the floats
      }
      *mine = __builtin_ldexpf(*mine, 127 - unit_found);
      if (lane == 0) units[step & 3] = unit_found;
    }
  };
  // 16 bits: K or V of the step that rows_at[at] was found for, into a slot
  auto dma_rows = [&](bool value, int at, int slot) {
    const uint8_t* base = (const uint8_t*)(value ? p.kv.v : p.kv.k);
    const uint32_t dst = lds0 + (uint32_t)((value ? S::V0 : 0) + slot * S::BYTES);
    const int64_t* rows = rows_at + at * 2 * kTileKeys + (value ? kTileKeys : 0) + dma_row;
    int64_t o[S::DMA];
    bool all = p.dim == HD;
#pragma unroll
    for (int i = 0; i < S::DMA; ++i) {
      o[i] = rows[i * ROWS1K];
      all = all && o[i] >= 0;
    }
    if (__builtin_amdgcn_ballot_w64(!all) == 0) {
      static_for<S::DMA>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        dma_load16_at(base + o[i] + (value ? v_off[i] : k_off[i]), dst, std::integral_constant<uint32_t, i * 1024>{});
      });
    } else {  // rows that are not there, and what lies past the head, are zeros
      static_for<S::DMA>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const uint32_t in_row = value ? v_off[i] : k_off[i];
        const void* src = o[i] >= 0 && in_row != kBufOOB ? (const void*)(base + o[i] + in_row) : (const void*)zero_piece;
        dma_load16_at(src, dst, std::integral_constant<uint32_t, i * 1024>{});
      });
    }
  };
  auto load_pieces = [&](bool value, int at) {
    const uint8_t* base = (const uint8_t*)(value ? p.kv.v : p.kv.k);
    int64_t o[PIECES];
    bool all = p.dim == HD;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      o[i] = rows_at[at * 2 * kTileKeys + (value ? kTileKeys : 0) + (i * 64 * NW + tid) / PPR];
      all = all && o[i] >= 0;
    }
    const int d = tid % PPR * EPP;
    if (__builtin_amdgcn_ballot_w64(!all) == 0) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) reg[i] = *(const u32x4_a8*)(base + o[i] + d * ES);
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        reg[i] = u32x4{0, 0, 0, 0};
        if (o[i] < 0 || d >= p.dim) continue;
        if (d + 8 >= p.dim) {  // the head ends in the middle of 16 codes
          const u32x2 h = *(const u32x2*)(base + o[i] + d);
          reg[i].x = h.x, reg[i].y = h.y;
        } else {
          reg[i] = *(const u32x4_a8*)(base + o[i] + d * ES);
        }
      }
    }
  };
  auto store_pieces = [&](bool value, int slot) {
    unsigned char* to = smem + (value ? S::V0 : 0) + slot * S::BYTES;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int n = i * 64 * NW + tid, r = n / PPR, c = (n % PPR) * (EPP / 8);
#pragma unroll
      for (int h = 0; h < EPP / 8; ++h) {
        const u32x2 a = e4m3x4<T>(reg[i][2 * h]), b = e4m3x4<T>(reg[i][2 * h + 1]);
        *(u32x4*)(to + (value ? v_place<HD>(r, 16 * (c + h)) : k_place<HD>(r, c + h))) = u32x4{a.x, a.y, b.x, b.y};
      }
    }
  };

  // ---- fragments: K's row `col` at chunk 2 kk + half (the second block of 32 keys lies a fixed
  // distance on), V's transposing reads: row 4 half + r16 / 4, columns 32 d + 16 (G % 2) +
  // 4 (r16 % 4) (further rows, multiples of 8, keep the permutation) ----
  int k_at[KK], v_at[DB];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) k_at[kk] = k_place<HD>(col, 2 * kk + half);
#pragma unroll
  for (int d = 0; d < DB; ++d)
    v_at[d] = S::V0 + v_place<HD>(4 * half + ((lane & 15) >> 2), 2 * (32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)));
  auto k_frag = [&](int slot, int n) {  // n: 2 kk + block
    return *(const u32x4*)(smem + k_at[n / 2] + slot * S::BYTES + (n & 1) * 32 * S::ROW);
  };
  auto v_frag = [&](int slot, int n) {  // n: g DB + d
    const unsigned char* at = smem + v_at[n % DB] + slot * S::BYTES + 16 * (n / DB) * S::ROW;
    const u32x2 lo = lds_read_tr(at), hi = lds_read_tr(at + 8 * S::ROW);
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };

  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x16{0};
  float m_ref = -INFINITY, sum = 0.f;
  float base = 0.f;                             // what is subtracted, in powers of two (0 for no key yet)
  const float unit = p.scale_log2;              // scores times this are powers of two
  // a weight is 2^TOP at the reference, and 2^(TOP + LAZY) at most before the reference is raised
  // (twice that with V's scale)
  constexpr float TOP = kHalf<T> ? 10.f : 0.f, LAZY = kHalf<T> ? 4.f : 8.f;
  int sum_unit = 127, step_unit = 127;  // of o, as `units`, and of the step's values
  u32x4 pw[4];                                  // weights of 16 keys each

  // scores of step j, before their maximum is taken: scales of 8-bit keys, keys that are not seen
  auto finish_scores = [&](f32x16 (&s)[2], int j) {
    const int key0 = key_of(j);
    if constexpr (k8) {
      const float* sc = scales + (j & 3) * 2 * kTileKeys + 4 * half;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const f32x4 c = *(const f32x4*)(sc + 32 * b + 2 * r);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[b][r + i] *= c[i];
        }
    }
    if (key0 + kTileKeys - 1 > wave_all) {
      const int most = limit - key0 - 4 * half;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 32 * b + 8 * (r / 4) + r % 4 <= most ? s[b][r] : -INFINITY;
    }
  };
  // with the maximum of a step's scores (of this lane's keys): the reference is raised
  auto raise = [&](float mx) {
    mx = max_halves(mx);
    if (__builtin_amdgcn_ballot_w64((mx - m_ref) * unit > LAZY)) {  // -inf - -inf is no reason
      const float m_new = fmaxf(m_ref, mx);
      const float alpha = m_new == m_ref ? 1.f : exp2_hw((m_ref - m_new) * unit);
      m_ref = m_new;
      base = m_new == -INFINITY ? 0.f : m_new * unit - TOP;
      sum *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
  };
  // pair t of a step's weights
  auto weigh = [&](f32x16 (&s)[2], int j, auto tc) {
    constexpr int t = decltype(tc)::value, b = t / 8, r = t % 8 * 2;
    float w0 = exp2_hw(__builtin_fmaf(s[b][r], unit, -base));
    float w1 = exp2_hw(__builtin_fmaf(s[b][r + 1], unit, -base));
    sum += w0 + w1;
    if constexpr (k8) {
      const float* sc = scales + (j & 3) * 2 * kTileKeys + kTileKeys + 4 * half + 32 * b + 8 * (r / 4) + r % 4;
      w0 *= sc[0];
      w1 *= sc[1];
    }
    uint32_t w = round2<T>(w0, w1);
    asm volatile("" : "+v"(w), "+v"(sum));  // computed here: not moved to where it is used
    pw[t / 4][t % 4] = w;
  };

  constexpr int AHEAD = 2;                 // fragments on their way from LDS (four, six: no faster)
  constexpr int N1 = 2 * KK, N2 = 4 * DB;  // products of the two phases
  constexpr int FIRST = 10;                // pairs of weights in the first phase (of 16), LEAD of them before
  constexpr int LEAD = 2;                  //   its first product, while that one's fragment arrives
  // step j: sc its scores, sn those of step j + 1 (past the last step whatever the slot holds, all
  // of it masked); f: fragments on their way
  auto first_phase = [&](int j, auto slotc, f32x16 (&sc)[2], f32x16 (&sn)[2], u32x4 (&f)[AHEAD]) {
    constexpr int slot = decltype(slotc)::value, next = slot ^ 1;
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) f[n] = k_frag(next, n);
    if constexpr (UNITS) step_unit = units[j & 3];
    sn[0] = sn[1] = f32x16{0};
    static_for<LEAD>([&](auto t) { weigh(sc, j, t); });
    __builtin_amdgcn_sched_barrier(0);
    static_for<N1>([&](auto nc) {
      constexpr int n = decltype(nc)::value;
      sn[n & 1] = Mfma32<T>::mma(f[n % AHEAD], q[n / 2], sn[n & 1]);
      if constexpr (n + AHEAD < N1) f[n % AHEAD] = k_frag(next, n + AHEAD);
      else f[n % AHEAD] = v_frag(slot, n + AHEAD - N1);
      static_for<FIRST - LEAD>([&](auto t) {
        if constexpr (decltype(t)::value * N1 / (FIRST - LEAD) == n)
          weigh(sc, j, std::integral_constant<int, LEAD + decltype(t)::value>{});
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    finish_scores(sn, j + 1);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto second_phase = [&](int j, auto slotc, f32x16 (&sc)[2], f32x16 (&sn)[2], u32x4 (&f)[AHEAD]) {
    constexpr int slot = decltype(slotc)::value;
    float mx = 0.f;
    if constexpr (UNITS) {
      const int to = __builtin_amdgcn_readfirstlane(step_unit);
      if (to != sum_unit) {
        const float by = __builtin_ldexpf(1.f, sum_unit - to);
        sum_unit = to;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= by;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // the other weights in the first half (groups 2 and 3 of 16 keys are used in the second), the
    // maximum in the second
    static_for<N2>([&](auto nc) {
      constexpr int n = decltype(nc)::value, HALF = N2 / 2;
      o[n % DB] = Mfma32<T>::mma(f[n % AHEAD], pw[n / DB], o[n % DB]);
      if constexpr (n + AHEAD < N2) f[n % AHEAD] = v_frag(slot, n + AHEAD);
      if constexpr (n < HALF) {
        static_for<16 - FIRST>([&](auto t) {
          if constexpr (decltype(t)::value * HALF / (16 - FIRST) == n)
            weigh(sc, j, std::integral_constant<int, FIRST + decltype(t)::value>{});
        });
      } else {
        static_for<16>([&](auto tc) {
          constexpr int t = decltype(tc)::value;
          if constexpr (t * HALF / 16 == n - HALF) {
            const float a = sn[t / 8][t % 8 * 2], b = sn[t / 8][t % 8 * 2 + 1];
            mx = t == 0 ? larger(a, b) : larger(mx, larger(a, b));
          }
        });
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    raise(mx);
  };
  static_assert(N1 % AHEAD == 0, "the fragments' places go on from one phase to the other");

  constexpr int STEP = KS * kTileKeys;  // keys from a step to the group's next one
  bool spoilt = false;
  if (KS > 1 && threadIdx.x == 0) any_spoilt = 0;
  if (turns > 0) {
    int page = -1;  // paged: of this thread's row, for the loads of the step after next
    if constexpr (!kPaged) {
      dma(false, 0, 0);
      dma(false, 1, 1);
      dma(true, 0, 0);
      ring_fence<2 * S::DMA>();  // K of step 0
    } else {
      const int key = key_of(0) + (tid & (kTileKeys - 1));
      place_row(0, key, page_number(key));  // K and V of step 0
      store_scale(0, 0);
      __syncthreads();
      find_unit(0);
      if constexpr (k8) {
        load_pieces(false, 0);
        store_pieces(false, 0);
        load_pieces(true, 0);
      } else {
        dma_rows(false, 0, 0);
        dma_rows(true, 0, 0);
      }
      const int k1 = key + STEP;
      place_row(1, k1, page_number(k1));  // K of step 1 (and V's scales of it)
      store_scale(1, 1);
      if constexpr (k8) store_pieces(true, 0);
      __syncthreads();
      if constexpr (k8)
        load_pieces(false, 1);
      else
        dma_rows(false, 1, 1);
      const int k2 = value_row ? k1 : k1 + STEP;
      place_row(0, k2, page_number(k2));  // K of step 2, V of step 1: for step 0's loads
      store_scale(2, 1);
      page = page_number(k2 + STEP);
      if constexpr (k8) store_pieces(false, 1);
      ring_fence<0>();
    }
    // the queries are here: else the compiler, which sees a path without their use, waits for them in
    // every step, and with them for the loads that the step has begun
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) asm volatile("" : "+v"(q[kk]));
    f32x16 s0[2], s1[2];
    if (key_of(0) <= wave_any) {
      s0[0] = s0[1] = f32x16{0};
#pragma unroll
      for (int n = 0; n < N1; ++n) {
        s0[n & 1] = Mfma32<T>::mma(k_frag(0, n), q[n / 2], s0[n & 1]);
        if (n % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      finish_scores(s0, 0);
      float mx = s0[0][0];
#pragma unroll
      for (int r = 1; r < 32; ++r) mx = larger(mx, s0[r / 16][r % 16]);
      raise(mx);
    }
    auto whole_step = [&](int j, auto slotc, f32x16 (&sc)[2], f32x16 (&sn)[2]) {
      constexpr int slot = decltype(slotc)::value;
      const int key0 = key_of(j);
      // K of step j + 1 and V of step j are in LDS; K of step j and V of step j - 1 are read
      ring_fence<0>();
      if constexpr (!kPaged) {
        dma(false, j + 2, slot);
        dma(true, j + 1, slot ^ 1);
      } else if constexpr (k8) {
        if (j + 1 < steps) load_pieces(false, slot);
      } else {
        asm volatile("" : "+v"(page));  // waited for here, not behind the loads that follow
        if (j + 1 < steps) {
          dma_rows(false, slot, slot);
          dma_rows(true, slot, slot ^ 1);
        }
      }
      if (begin + (j + 1) * STEP - 1 > tile_all) {  // of any of the groups: all waves come here
        unsigned char* vs = smem + S::V0 + slot * S::BYTES;
        bool bad = false;  // a group's waves find the same
        if (key0 + kTileKeys - 1 > tile_all) {
          bad = any_not_finite<T>(vs, S::BYTES);
          if constexpr (k8) bad = bad || __builtin_amdgcn_ballot_w64(not_finite(value_scales(j)[lane])) != 0;
        }
        if (KS > 1 || bad) {
          __syncthreads();
          if (bad) {
            spoilt = true;
            if (KS > 1) any_spoilt = 1;
            for (int i = 16 * tid; i < S::BYTES; i += 16 * 64 * NW) *(u32x4*)(vs + i) = finite_only<T>(*(const u32x4*)(vs + i));
            if (k8 && wave == 0 && not_finite(value_scales(j)[lane])) value_scales(j)[lane] = 0.f;
          }
          __syncthreads();
        }
      }
      u32x4 f[AHEAD];
      const bool active = key0 <= wave_any;
      if (active) first_phase(j, slotc, sc, sn, f);
      if constexpr (kPaged) {
        if (j + 1 < steps) {
          if constexpr (k8) {
            find_unit(j + 1);
            store_pieces(false, slot);
            load_pieces(true, slot);
          }
          const int key = key0 + (value_row ? 2 : 3) * STEP + (tid & (kTileKeys - 1));
          place_row(slot ^ 1, key, page);
          page = page_number(key + STEP);
        }
      }
      if (active) second_phase(j, slotc, sc, sn, f);
      if constexpr (k8) {
        if (j + 1 < steps) {
          store_pieces(true, slot ^ 1);
          store_scale(j + 3, j + 2);
        }
      }
    };
    // a step's scores change places with the next one's
    for (int j = 0; j < turns; j += 2) {
      whole_step(j, std::integral_constant<int, 0>{}, s0, s1);
      if (j + 1 < turns) whole_step(j + 1, std::integral_constant<int, 1>{}, s1, s0);
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // no LDS DMA may outlive its slot's use, or the workgroup
  }
  if constexpr (UNITS) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = __builtin_ldexpf(o[d][r], sum_unit - 127);
  }

  if (KS > 1) {
    __syncthreads();
    spoilt = any_spoilt != 0;
  }
  if (spoilt) {  // add what was made zero (see any_not_finite)
    for (int j = 0; j < turns; ++j) {
      const int key0 = key_of(j);
      if (begin + (j + 1) * STEP - 1 <= tile_all) continue;
      ring_fence<0>();  // V's first slot is read
      if constexpr (!kPaged) {
        dma(true, j, 0);
      } else {
        const int key = key0 + (tid & (kTileKeys - 1));
        const int page = page_number(key);
        place_row(0, key, page);
        if constexpr (k8) {
          if (wave == 1) {
            // where the scales are is read again: kept through the loop for this, it costs registers (129.5 us for
            // 125.9, 4 chunks of up to 512 over up to 8100 keys, heads 32 / 8 of 128)
            auto args = (const __attribute__((address_space(4))) AttnParams*)__builtin_amdgcn_kernarg_segment_ptr();
            asm("" : "+s"(args));
            const int place = key % args->kv.page_size;
            float s = 0.f;
            if ((unsigned)page < (unsigned)args->kv.pages)
              s = args->kv.v_scale[page * args->kv.vs_page + place * args->kv.vs_token + kvh * args->kv.vs_head];
            value_scales(0)[lane] = s;
          }
        }
        __syncthreads();
        if constexpr (k8) {
          load_pieces(true, 0);
          store_pieces(true, 0);
          __syncthreads();
          const float* sc = value_scales(0);
          for (int i = 16 * tid; i < S::BYTES; i += 16 * 64 * NW) {
            const int r = i / S::ROW;  // v_place keeps to its row
            u32x4* at = (u32x4*)(smem + S::V0 + i);
            if (not_finite(sc[r])) *at = times<T>(*at, sc[r]);
          }
        } else {
          dma_rows(true, 0, 0);
        }
      }
      ring_fence<0>();
      if (key0 + kTileKeys - 1 <= tile_all) continue;  // this group's step was left as it is
      for (int kind = 0; kind < 3; ++kind)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          f32x16 hit = f32x16{0};
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int key = key0 + 16 * g + 4 * half;
            const u32x4 seen = {ones_up_to<T>(key, limit), ones_up_to<T>(key + 2, limit), ones_up_to<T>(key + 8, limit),
                                ones_up_to<T>(key + 10, limit)};
            hit = Mfma32<T>::mma(kind_ones<T>(v_frag(0, g * DB + d), kind), seen, hit);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] += hit[r] > 0.f ? kind_value(kind) : 0.f;
        }
    }
  }

  if constexpr (KS == 2) {  // the second group's sums to the first, lane by lane
    f32x4* to = (f32x4*)all_smem;
    float* ml = (float*)(to + DB * 4 * 64 * NW);
    static_assert(S::LDS * KS >= DB * 4 * 64 * NW * 16 + 64 * NW * 8, "LDS");
    __syncthreads();
    if (part_k == 1) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          to[(4 * d + r / 4) * 64 * NW + tid] = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
      ml[tid] = m_ref;
      ml[64 * NW + tid] = sum;
    }
    __syncthreads();
    if (part_k == 0) {
      const float m1 = ml[tid], m = fmaxf(m_ref, m1);
      const float a0 = m_ref == m ? 1.f : exp2_hw((m_ref - m) * unit), a1 = m1 == m ? 1.f : exp2_hw((m1 - m) * unit);
      sum = sum * a0 + ml[64 * NW + tid] * a1;
      m_ref = m;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const f32x4 x = to[(4 * d + r / 4) * 64 * NW + tid];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][r + i] = o[d][r + i] * a0 + x[i] * a1;
        }
    }
  }

  // ---- out: lane has row `out_row`, elements 32 d + 8 (r / 4) + 4 half + r % 4 ----
  __syncthreads();
  Seq os;
  os.b = __builtin_amdgcn_readfirstlane(kept_seq.b);
  os.q0 = __builtin_amdgcn_readfirstlane(kept_seq.q0);
  os.len_q = __builtin_amdgcn_readfirstlane(kept_seq.len_q);
  os.len_k = __builtin_amdgcn_readfirstlane(kept_seq.len_k);
  const int out_kvh = __builtin_amdgcn_readfirstlane(kept_kvh), out_row0 = __builtin_amdgcn_readfirstlane(kept_row0);
  const int out_splits = __builtin_amdgcn_readfirstlane(kept_splits);
  const int out_row = out_row0 + wave * 32 + col, out_rows = os.len_q * p.group;
  sum += __shfl_xor(sum, 32);
  if (out_splits > 1) {
    float* part = part_of_tile(p, BM);
    if (out_row < out_rows && part_k == 0) {
      const uint32_t at = part_at(p, BM, blockIdx.y);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int e = 32 * d + 8 * (r / 4) + 4 * half;
          if (e < p.dim)
            store16_coherent(part, at + part_o(p, out_row - out_row0) + 4 * e, f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]});
        }
      if (half == 0) store8_coherent(part, at + part_ml(p, BM, out_row - out_row0), m_ref * unit, sum);
    }
    join_if_last<T, 64 * NW * KS>(p, os, out_kvh, out_row0, min(BM, out_rows - out_row0), part, BM, out_splits, all_smem);
    return;
  }
  if (out_row >= out_rows || part_k != 0) return;
  const float inv = row_factor(p, os, out_row, sum);
  const int out_tok = out_row / p.group, out_head = out_kvh * p.group + out_row - out_tok * p.group;
  T* op = (T*)p.out + os.b * p.out_batch + (int64_t)(os.q0 + out_tok) * p.out_token + (int64_t)out_head * p.out_head;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int e = 32 * d + 8 * (r / 4) + 4 * half;
      if (e < p.dim)
        *(u32x2*)(op + e) = u32x2{round2<T>(o[d][r] * inv, o[d][r + 1] * inv), round2<T>(o[d][r + 2] * inv, o[d][r + 3] * inv)};
    }
}

// hd: the padded head; ks: groups of a workgroup, 2 for hd up to 128 only.
template <typename T, int KIND>
hipError_t launch_tile_hd(int hd, int ks, const AttnParams& p, dim3 grid, hipStream_t s) {
  const dim3 block(64 * kTileWaves * ks);
  if (hd == 256) return launch_kernel(attention_tile_kernel<T, 256, KIND, 1>, grid, block, 0, s, p);
  if (ks == 2)
    return hd == 64 ? launch_kernel(attention_tile_kernel<T, 64, KIND, 2>, grid, block, 0, s, p)
                    : launch_kernel(attention_tile_kernel<T, 128, KIND, 2>, grid, block, 0, s, p);
  return hd == 64 ? launch_kernel(attention_tile_kernel<T, 64, KIND, 1>, grid, block, 0, s, p)
                  : launch_kernel(attention_tile_kernel<T, 128, KIND, 1>, grid, block, 0, s, p);
}

}  // namespace cmpext3
