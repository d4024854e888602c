// Attention of few query rows over a paged cache (gfx950): generation, bound by reading the
// cache.
//
// Rows: a workgroup takes 16 MB rows of one sequence and one kv head (row r: query
// r / group, head r % group), so that one pass over the cache serves the whole group of
// heads, and one range of keys (split_keys of them); its four waves (eight for short 8-bit keys)
// take steps of 32 keys in turn, each with a running maximum and sum of its own, and are joined at
// the end in LDS.  The ranges are joined as attention_join.h says, if there is more than one.
//
// Products (16x16x32, fp32 sums) run transposed as in the tile kernel: S^T = K Q^T with the
// keys' fragments loaded straight from the cache into registers (a lane's 16 bytes are one
// fragment; 8-bit codes are two, the head's elements then taken in another order by both
// operands), O^T = V^T P^T with V through a stretch of LDS that only this wave uses, and
// transposing reads.  Each step's loads start when the step before has used its registers, and
// its page numbers, one per lane, are fetched another step ahead.  A weight is taken as the sum
// of two 16-bit numbers (the second product twice): there is time for it under the loads (188.5 us
// below with and without), and the result is then off by its own rounding only.  Over codes the
// weight carries its value's scale, which may be any float: the two numbers are bf16 there whatever
// the queries are (16 bits of a weight together, and codes fit bf16 as well), as fp16 ends at 2^-25
// (4096 keys with values of size 1e-3: off by 6e-4, which is the result's own rounding, in fp16 by 1e-2).
//
// MI355X, heads 32 / 8 of 128: 64 sequences of up to 8192 keys in 16 bits, 875 MB, 188 us (4.65 TB/s;
// a large copy moves 5.25): two workgroups a CU, 16 KB of each wave on their way.  One of 65537 keys
// in 8 bits, 138 MB, 39 us: the scales, 4 bytes of each 32, are fetched by every XCD (169 MB read),
// and starting, joining 57 splits and launching take about 10.  Steps of 64 keys of 8 bits, with two
// waves on a SIMD for three, took 43; loads past the caches' reusable lines 42 (and 195 in 16 bits).
#pragma once

#include "attention_join.h"

namespace cmpext3 {

template <int HD, int MB, int NW>
struct FewShape {
  static constexpr int BM = 16 * MB;
  static constexpr int V_BYTES = kWaveKeys * HD * 2;
  // V, the scales of K and V, the byte offsets of the keys' and values' rows in the cache
  static constexpr int WAVE = V_BYTES + 2 * kWaveKeys * 4 + 2 * kWaveKeys * 8;
  static constexpr int PITCH = HD + 4;                      // floats of a row of O in LDS
  static constexpr int JOIN = NW * BM * PITCH * 4;
  static constexpr int ML = NW * BM * 2 * 4;
  static constexpr int BODY = WAVE * NW > JOIN ? WAVE * NW : JOIN;
  static constexpr int LDS = BODY + ML > kJoinBytes ? BODY + ML : kJoinBytes;
};

// Byte offset of byte column `bc` of V's row `row`: a transposing read by 32 lanes covers
// eight rows of 32 bytes, which fall on all banks once.
template <int HD>
__device__ __forceinline__ int few_v_place(int row, int bc) {
  if constexpr (HD == 64)
    return row * 128 + (((bc >> 5) ^ ((row >> 1) & 3)) << 5) + (bc & 31);
  else
    return row * HD * 2 + (((bc >> 6) ^ (row & 3)) << 6) + ((bc & 63) ^ (((row >> 2) & 1) << 5));
}

// The waves a SIMD holds at least: as many as have registers; of eight waves (NW) one workgroup is enough.
template <typename T, int HD, int KIND, int MB, int NW>
__global__ void __launch_bounds__(64 * NW, HD == 256 ? 1 : MB == 2 || NW == 8 ? 2 : HD == 64 ? 4 : KIND == kKvPaged8 ? 3 : 2) attention_few_kernel(const AttnParams p) {
  constexpr bool k8 = KIND == kKvPaged8;
  using W = std::conditional_t<k8, __bf16, T>;  // the second product's operands
  using S = FewShape<HD, MB, NW>;
  constexpr int KK = HD / 32, DB = HD / 16;
  constexpr int EPP = k8 ? 16 : 8, ES = k8 ? 1 : 2;
  constexpr int KN = HD / (4 * EPP);              // 16-byte loads of a lane for a block of 16 keys
  constexpr int PPR = HD / EPP, VN = kWaveKeys * PPR / 64;
  __shared__ __attribute__((aligned(16))) unsigned char smem[S::LDS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, G = lane >> 4;
  const int kvh = blockIdx.x % p.kv_heads;
  const Seq sq = seq_of_slot(p, blockIdx.x / p.kv_heads, S::BM);
  if (sq.b < 0) return;
  const int split = blockIdx.y;
  const int shift = sq.len_k - sq.len_q;
  const int row0 = sq.tile * S::BM, rows = sq.len_q * p.group;
  int end = keys_end(p, sq, min(row0 + S::BM, rows) - 1);
  const int splits = NW == 8 ? 1 : splits_of(p, sq, end);  // eight waves take whole keys
  if (split >= splits) return;
  const int begin = split * p.split_keys;
  end = min(end, begin + p.split_keys);

  // keys up to `all` are seen by every row of the tile
  const int all = p.causal ? min(row0 / p.group + shift, sq.len_k - 1) : sq.len_k - 1;
  int limit[MB];
  u32x4 q[MB][KK];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int row = row0 + 16 * mb + r16;
    const int tok = min(row, rows - 1) / p.group, head = kvh * p.group + min(row, rows - 1) - tok * p.group;
    limit[mb] = p.causal ? min(tok + shift, sq.len_k - 1) : sq.len_k - 1;
    const T* qp = (const T*)p.q + sq.b * p.q_batch + (int64_t)(sq.q0 + tok) * p.q_token + (int64_t)head * p.q_head;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = k8 ? 64 * (kk / 2) + 16 * G + 8 * (kk & 1) : 32 * kk + 8 * G;
      q[mb][kk] = row < rows && d < p.dim ? *(const u32x4*)(qp + d) : u32x4{0, 0, 0, 0};
    }
  }

  unsigned char* vs = smem + wave * S::WAVE;
  float* sc = (float*)(vs + S::V_BYTES);
  const int32_t* table = p.kv.table + sq.b * p.kv.table_row;
  const uint8_t* kc = (const uint8_t*)p.kv.k;
  const uint8_t* vc = (const uint8_t*)p.kv.v;

  // ---- loads of a step: lane l < 32 looks after key l's row of K, lane 32 + l after V's ----
  int64_t* row_at = (int64_t*)(sc + 2 * kWaveKeys);
  const bool value = lane >= kWaveKeys;
  const int64_t c_page = value ? p.kv.v_page : p.kv.k_page, c_token = value ? p.kv.v_token : p.kv.k_token;
  const int64_t c_head = kvh * (value ? p.kv.v_head : p.kv.k_head);
  const float* c_scale = k8 ? (value ? p.kv.v_scale + kvh * p.kv.vs_head : p.kv.k_scale + kvh * p.kv.ks_head) : nullptr;
  const int64_t s_page = value ? p.kv.vs_page : p.kv.ks_page, s_token = value ? p.kv.vs_token : p.kv.ks_token;
  const int my_key = lane & (kWaveKeys - 1);
  // the page of this lane's key of a step, as far as the table goes; fetched a step ahead
  auto page_number = [&](int key0) -> int {
    const int key = key0 + my_key, n = p.kv.page_shift >= 0 ? key >> p.kv.page_shift : key / p.kv.page_size;
    return n < p.kv.table_pages ? table[n] : -1;
  };
  u32x4 kr[2][KN], vr[VN];
  float sr = 0.f;
  // 16 bytes at element d of a row (8 where the head ends in the middle of 16 codes)
  auto piece = [&](const uint8_t* at, int d) -> u32x4 {
    if (k8 && d + 8 >= p.dim) {
      const u32x2 h = *(const u32x2*)(at + d);
      return u32x4{h.x, h.y, 0, 0};
    }
    return *(const u32x4_a8*)(at + d * ES);
  };
  auto load = [&](int key0, int page) {
    const int key = key0 + my_key;
    const int place = p.kv.page_shift >= 0 ? key & (p.kv.page_size - 1) : key % p.kv.page_size;
    const bool there = key < sq.len_k && (unsigned)page < (unsigned)p.kv.pages;
    row_at[lane] = there ? (page * c_page + place * c_token + c_head) * ES : -1;
    if constexpr (k8) {
      sr = 0.f;
      if (there) sr = c_scale[page * s_page + place * s_token];
    }
    if (__builtin_amdgcn_ballot_w64(!there) == 0 && p.dim == HD) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint8_t* at = kc + row_at[16 * b + r16];
#pragma unroll
        for (int i = 0; i < KN; ++i) kr[b][i] = *(const u32x4_a8*)(at + (4 * EPP * i + EPP * G) * ES);
      }
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const int n = i * 64 + lane;
        vr[i] = *(const u32x4_a8*)(vc + row_at[kWaveKeys + n / PPR] + (n % PPR) * EPP * ES);
      }
    } else {  // rows that are not there, and what lies past the head, are zeros
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int64_t at = row_at[16 * b + r16];
#pragma unroll
        for (int i = 0; i < KN; ++i) {
          const int d = 4 * EPP * i + EPP * G;
          kr[b][i] = u32x4{0, 0, 0, 0};
          if (at >= 0 && d < p.dim) kr[b][i] = piece(kc + at, d);
        }
      }
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const int n = i * 64 + lane, d = (n % PPR) * EPP;
        const int64_t at = row_at[kWaveKeys + n / PPR];
        vr[i] = u32x4{0, 0, 0, 0};
        if (at >= 0 && d < p.dim) vr[i] = piece(vc + at, d);
      }
    }
  };

  f32x4 o[MB][DB];
  float m_ref[MB], sum[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    m_ref[mb] = -INFINITY;
    sum[mb] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[mb][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float unit = k8 ? 1.f : p.scale_log2;
  constexpr float TOP = kHalf<W> ? 15.f : 0.f;  // the largest weight is 2^TOP (see kHalf)

  // V of a step into this wave's LDS, and its fragments from there: keys 4 G .. and 16 + 4 G ..
  auto store_v = [&]() {
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      const int n = i * 64 + lane, r = n / PPR, c = (n % PPR) * EPP * 2;
      if constexpr (k8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x2 a = e4m3x4<W>(vr[i][2 * h]), b = e4m3x4<W>(vr[i][2 * h + 1]);
          *(u32x4*)(vs + few_v_place<HD>(r, c + 16 * h)) = u32x4{a.x, a.y, b.x, b.y};
        }
      } else {
        *(u32x4*)(vs + few_v_place<HD>(r, c)) = vr[i];
      }
    }
  };
  auto v_frag = [&](int d) {
    const int row = 4 * G + (r16 >> 2), bc = 2 * (16 * d + 4 * (r16 & 3));
    const u32x2 lo = lds_read_tr(vs + few_v_place<HD>(row, bc));
    const u32x2 hi = lds_read_tr(vs + few_v_place<HD>(row + 16, bc));
    return u32x4{lo.x, lo.y, hi.x, hi.y};
  };

  constexpr int STEP = NW * kWaveKeys;
  // values that are not finite are looked for in steps with keys past this, and added in a second pass over those
  // (all of them once a scale is not finite: what a step has had already it gets again, infinity or NaN)
  int whole = all;
  bool spoilt = false;
  int key0 = begin + wave * kWaveKeys;
  int page = -1;
  if (key0 < end) {
    load(key0, page_number(key0));
    page = page_number(key0 + STEP);
  }
  for (; key0 < end; key0 += STEP) {
    store_v();
    if constexpr (k8) {
      const bool bad = value && not_finite(sr);
      if (__builtin_amdgcn_ballot_w64(bad) != 0) {
        spoilt = true;
        whole = -1;
        if (bad) sr = 0.f;
      }
      sc[lane] = sr;
    }
    __builtin_amdgcn_sched_barrier(0);  // V's registers are free
    f32x4 s[MB][2];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) s[mb][0] = s[mb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        u32x4 k;
        if constexpr (k8) {
          const u32x2 lo = e4m3x4<T>(kr[b][kk / 2][2 * (kk & 1)]), hi = e4m3x4<T>(kr[b][kk / 2][2 * (kk & 1) + 1]);
          k = u32x4{lo.x, lo.y, hi.x, hi.y};
        } else {
          k = kr[b][kk];
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) s[mb][b] = Mfma<T>::mma(k, q[mb][kk], s[mb][b]);
      }
    __builtin_amdgcn_sched_barrier(0);  // and K's
    if (key0 + STEP < end) {
      load(key0 + STEP, page);
      page = page_number(key0 + 2 * STEP);
    }
    f32x4 ksc[2], vsc[2];
    if constexpr (k8) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        ksc[b] = *(const f32x4*)(sc + 16 * b + 4 * G);
        vsc[b] = *(const f32x4*)(sc + 32 + 16 * b + 4 * G);
      }
    }
    u32x4 pw[MB], pl[MB];  // weights, and what cutting them left
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 16 * b + 4 * G + i;
          float x = s[mb][b][i];
          if constexpr (k8) x *= ksc[b][i] * p.scale_log2;
          x = key <= limit[mb] && key < end ? x : -INFINITY;
          s[mb][b][i] = x;
          mx = fmaxf(mx, x);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m_ref[mb], mx);
      if (__builtin_amdgcn_ballot_w64(m_new != m_ref[mb])) {
        const float alpha = m_new == m_ref[mb] ? 1.f : exp2_hw((m_ref[mb] - m_new) * unit);
        m_ref[mb] = m_new;
        sum[mb] *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[mb][d] *= alpha;
      }
      const float base = m_ref[mb] == -INFINITY ? 0.f : m_ref[mb] * unit - TOP;
      float w[8];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = exp2_hw(k8 ? s[mb][b][i] - base : __builtin_fmaf(s[mb][b][i], unit, -base));
          sum[mb] += x;
          w[4 * b + i] = k8 ? x * vsc[b][i] : x;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pw[mb][i] = cut2<W>(w[2 * i], w[2 * i + 1]);
        pl[mb][i] = rest2<W>(w[2 * i], w[2 * i + 1], pw[mb][i]);
      }
    }
    if (key0 + kWaveKeys - 1 > whole && any_not_finite<W>(vs, S::V_BYTES)) {
      spoilt = true;
      for (int i = 16 * lane; i < S::V_BYTES; i += 1024) *(u32x4*)(vs + i) = finite_only<W>(*(const u32x4*)(vs + i));
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const u32x4 v = v_frag(d);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) o[mb][d] = Mfma<W>::mma(v, pl[mb], Mfma<W>::mma(v, pw[mb], o[mb][d]));
      if (d % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (spoilt) {  // add what was made zero (see any_not_finite)
    for (key0 = begin + wave * kWaveKeys; key0 < end; key0 += STEP) {
      if (key0 + kWaveKeys - 1 <= whole) continue;
      load(key0, page_number(key0));
      store_v();
      if constexpr (k8) {
        const unsigned long long bad = __builtin_amdgcn_ballot_w64(value && not_finite(sr)) >> kWaveKeys;
        sc[lane] = sr;
        for (int i = 16 * lane; bad != 0 && i < S::V_BYTES; i += 1024) {
          const int r = i / (2 * HD);  // few_v_place keeps to its row
          if (bad >> r & 1) *(u32x4*)(vs + i) = times<W>(*(const u32x4*)(vs + i), sc[kWaveKeys + r]);
        }
      }
      for (int kind = 0; kind < 3; ++kind)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const int key = key0 + 4 * G, most = min(limit[mb], end - 1);
          const u32x4 seen = {ones_up_to<W>(key, most), ones_up_to<W>(key + 2, most), ones_up_to<W>(key + 16, most),
                              ones_up_to<W>(key + 18, most)};
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const f32x4 hit = Mfma<W>::mma(kind_ones<W>(v_frag(d), kind), seen, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i) o[mb][d][i] += hit[i] > 0.f ? kind_value(kind) : 0.f;
          }
        }
    }
  }

  // ---- join the waves ----
  float* ml = (float*)(smem + S::BODY);         // [wave][row][2]
  __syncthreads();                              // every wave is done with its stretch of LDS
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    sum[mb] += __shfl_xor(sum[mb], 16);
    sum[mb] += __shfl_xor(sum[mb], 32);
    const int r = 16 * mb + r16;
    if (G == 0) {
      ml[(wave * S::BM + r) * 2] = m_ref[mb] * unit;
      ml[(wave * S::BM + r) * 2 + 1] = sum[mb];
    }
    float* po = (float*)smem + (wave * S::BM + r) * S::PITCH;
#pragma unroll
    for (int d = 0; d < DB; ++d) *(f32x4*)(po + 16 * d + 4 * G) = o[mb][d];
  }
  __syncthreads();
  constexpr int QUADS = HD / 4;
  float* part = part_of_tile(p, S::BM);
  for (int n = tid; n < S::BM * QUADS; n += 64 * NW) {
    const int r = n / QUADS, e = (n % QUADS) * 4, row = row0 + r;
    if (row >= rows || e >= p.dim) continue;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, ml[(w * S::BM + r) * 2]);
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = m == -INFINITY ? 0.f : exp2_hw(ml[(w * S::BM + r) * 2] - m);  // times a sum of NaN: still NaN
      l += f * ml[(w * S::BM + r) * 2 + 1];
      acc += f * *(const f32x4*)((const float*)smem + (w * S::BM + r) * S::PITCH + e);
    }
    if (splits > 1) {
      store16_coherent(part, part_at(p, S::BM, split) + part_o(p, r) + 4 * e, acc);
      if (e == 0) store8_coherent(part, part_at(p, S::BM, split) + part_ml(p, S::BM, r), m, l);
    } else {
      const int tok = row / p.group, head = kvh * p.group + row - tok * p.group;
      const float inv = row_factor(p, sq, row, l);
      T* op = (T*)p.out + sq.b * p.out_batch + (int64_t)(sq.q0 + tok) * p.out_token + (int64_t)head * p.out_head;
      *(u32x2*)(op + e) = u32x2{round2<T>(acc[0] * inv, acc[1] * inv), round2<T>(acc[2] * inv, acc[3] * inv)};
    }
  }
  if (splits > 1) join_if_last<T, 64 * NW>(p, sq, kvh, row0, min(S::BM, rows - row0), part, S::BM, splits, smem);
}

// waves: 4, or 8 for 8 bits, 16 rows and hd up to 128.
template <typename T, int KIND, int MB>
hipError_t launch_few_hd(int hd, int waves, const AttnParams& p, dim3 grid, hipStream_t s) {
  const dim3 block(64 * waves);
  if constexpr (MB == 1 && KIND == kKvPaged8) {
    if (waves == 8)
      return hd == 64 ? launch_kernel(attention_few_kernel<T, 64, KIND, 1, 8>, grid, block, 0, s, p)
                      : launch_kernel(attention_few_kernel<T, 128, KIND, 1, 8>, grid, block, 0, s, p);
  }
  if (hd == 64) return launch_kernel(attention_few_kernel<T, 64, KIND, MB, 4>, grid, block, 0, s, p);
  if (hd == 128) return launch_kernel(attention_few_kernel<T, 128, KIND, MB, 4>, grid, block, 0, s, p);
  if constexpr (MB == 1) return launch_kernel(attention_few_kernel<T, 256, KIND, MB, 4>, grid, block, 0, s, p);
  return hipErrorInvalidValue;  // heads over 128 take 16 rows: two blocks' sums do not fit the registers
}

}  // namespace cmpext3
