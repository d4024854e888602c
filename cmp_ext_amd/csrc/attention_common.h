// Device helpers of the attention operators: where a sequence's rows and keys are,
// page lookups, and 8-bit floats.
#pragma once

#include "attention_params.h"
#include "device_common.h"

namespace cmpext3 {

// One sequence of a call.
struct Seq {
  int b;           // -1: none
  int q0, len_q;   // first row in the packed queries, number of queries
  int k0, len_k;
  int tile;        // row tile of the sequence
  int split_keys;  // keys of a split
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Keys of a paged sequence: its length, as far as the table goes.
__device__ __forceinline__ int paged_keys(const AttnParams& p, int seq_len) {
  return (int)min((int64_t)max(seq_len, 0), (int64_t)p.kv.table_pages * p.kv.page_size);
}

// Sum of x over this lane and those below it.
__device__ __forceinline__ int sum_below(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // 1, 2, 4 and 8 lanes below, in rows of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row 0 to row 1, 2 to 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // the lower half to the upper
  return x;
}

// The largest x of all lanes.
__device__ __forceinline__ int largest(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xf, 0xf, false));  // as in sum_below
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}

// Keys of a split, a multiple of 128, such that all tiles' splits are p.fit workgroups at most: the
// least such number that p.split_keys and p.splits allow; all keys, if there is none.  Lane e has
// entry e's queries and keys (seq_of_slot).  All workgroups find the same.
__device__ __forceinline__ int fitting_split(const AttnParams& p, int rows, int len_q, int len_k) {
  const int t = (threadIdx.x & 63) < p.batch + 2 && len_k > 0 ? (len_q * p.group + rows - 1) / rows : 0;
  const int longest = (largest(t > 0 ? len_k : 0) + 127) / 128;
  int low = max(p.split_keys / 128, (longest + p.splits - 1) / p.splits), high = max(longest, low);  // in 128 keys
  while (low < high) {
    const int mid = (low + high) / 2, keys = 128 * mid;
    if (__builtin_amdgcn_readlane(sum_below(t * ((len_k + keys - 1) / keys)), 63) * p.kv_heads <= p.fit)
      high = mid;
    else
      low = mid + 1;
  }
  return 128 * high;
}

// Row tile `slot` in the order of the keys the tiles see, most first, over all of up to 62 sequences:
// the sequence's entry e (seq_of_slot) and its tile; e = -1 past the last tile.  Lane e has entry e's
// queries and keys.  With cost c(i) = max(0, i + 1 + off) of tile i of t (causal, off the keys before
// its first query, in tiles; else the same for all), the tiles that cost L or more are
//   n(L) = clamp(t + off - L + 1, 0, t)
// of an entry; the wanted level is the last with more than `slot` of them in all.
__device__ __forceinline__ int longest_first(const AttnParams& p, int slot, int rows, int len_q, int len_k, int& tile) {
  const int lane = threadIdx.x & 63;
  const int t = lane < p.batch + 2 ? (len_q * p.group + rows - 1) / rows : 0;
  const int per = max(1, rows / p.group);  // queries of a tile
  // the cost of the last tile
  const int h = t == 0 || len_k == 0 ? 0 : p.causal ? t + (len_k - len_q) / per : len_k / per + 1;
  auto at_least = [&](int level) { return level <= 0 ? t : p.causal ? clampi(h - level + 1, 0, t) : level <= h ? t : 0; };
  if (__builtin_amdgcn_readlane(sum_below(t), 63) <= slot) return -1;
  int low = 0;
  for (int step = 1 << 30; step > 0; step >>= 1) {
    if (__builtin_amdgcn_ballot_w64(h >= low + step) == 0) continue;
    if (__builtin_amdgcn_readlane(sum_below(at_least(low + step)), 63) > slot) low += step;
  }
  const int above = at_least(low + 1), here = at_least(low) - above;
  const int before = __builtin_amdgcn_readlane(sum_below(above), 63);
  const int upto = before + sum_below(here);
  const int e = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > slot));
  const int te = __builtin_amdgcn_readlane(t, e), he = __builtin_amdgcn_readlane(h, e);
  const int r = slot - (__builtin_amdgcn_readlane(upto, e) - __builtin_amdgcn_readlane(here, e));
  tile = clampi(low > 0 && p.causal ? low - 1 - he + te : r, 0, max(te - 1, 0));
  return e;
}

// The sequence that holds row tile `slot` of the grid, and which of its tiles of `rows` rows that is
// (a row is one query of one head of the group).  With packed queries, the rows before the first
// sequence and those past the last one count as sequences without keys, e = 0 and batch + 1 (zeros
// go out), sequence b as e = b + 1; e owns the slots from (its first query) * group / rows + e on: these
// grow by at least one per sequence and by no less than its tiles, so the grid needs no lengths
// from the host; slots past a sequence's last tile have nothing to do (b = -1).  Each lane looks
// at one sequence, 64 at a time, and loads all that is known of it at once: what follows waits for
// one memory access, not for three in a row.  SORTED: p.longest_first may be set (paged keys).
template <bool SORTED = false>
__device__ __forceinline__ Seq seq_of_slot(const AttnParams& p, int slot, int rows) {
  Seq s;
  s.split_keys = p.split_keys;
  int start_k = 0, end_k = p.len_k;  // or, paged, the length as end_k
  if (p.starts_q == nullptr) {
    const int tiles = (p.len_q * p.group + rows - 1) / rows;
    s.b = slot / tiles;
    s.tile = slot - s.b * tiles;
    s.q0 = 0;
    s.len_q = p.len_q;
    if (p.kv.table != nullptr) {
      end_k = p.seq_lens[s.b];
    } else if (p.starts_k != nullptr) {
      start_k = p.starts_k[s.b];
      end_k = p.starts_k[s.b + 1];
    }
  } else {
    const int lane = threadIdx.x & 63;
    int at = -1, first = 0, q_from = 0, q_to = 0, k_from = 0, k_to = 0;
    for (int e0 = 0; e0 < p.batch + 2; e0 += 64) {
      const int e = min(e0 + lane, p.batch + 1), b = clampi(e - 1, 0, max(p.batch - 1, 0));
      int from = p.starts_q[max(e - 1, 0)], to = p.starts_q[min(e, p.batch)];
      int kf = 0, kt = p.len_k;
      if (p.batch > 0) {
        if (p.kv.table != nullptr) {
          kt = p.seq_lens[b];
        } else if (p.starts_k != nullptr) {
          kf = p.starts_k[b];
          kt = p.starts_k[b + 1];
        }
      }
      if (e == 0) from = 0, kf = kt = 0;
      if (e == p.batch + 1) to = p.total_q, kf = kt = 0;
      const int q = clampi(from, 0, p.total_q);
      const bool below = e0 + lane < p.batch + 2 && q * p.group / rows + e <= slot;
      const unsigned long long m = __builtin_amdgcn_ballot_w64(below);
      const int n = __builtin_popcountll(m);
      if (n > 0) {
        at = n - 1;
        first = e0;
        q_from = q, q_to = to, k_from = kf, k_to = kt;
      }
      if (n < 64) break;
    }
    if constexpr (SORTED) {
      if (p.fit > 0) s.split_keys = fitting_split(p, rows, clampi(q_to, q_from, p.total_q) - q_from, paged_keys(p, k_to));
      if (p.longest_first) {
        at = longest_first(p, slot, rows, clampi(q_to, q_from, p.total_q) - q_from, paged_keys(p, k_to), s.tile);
        s.b = -1;
        if (at < 0) return s;
      }
    }
    s.q0 = __builtin_amdgcn_readlane(q_from, at);
    s.len_q = clampi(__builtin_amdgcn_readlane(q_to, at), s.q0, p.total_q) - s.q0;
    if (!SORTED || !p.longest_first) s.tile = slot - (s.q0 * p.group / rows + first + at);
    s.b = clampi(first + at - 1, 0, max(p.batch - 1, 0));
    start_k = __builtin_amdgcn_readlane(k_from, at);
    end_k = __builtin_amdgcn_readlane(k_to, at);
  }
  s.b = __builtin_amdgcn_readfirstlane(s.b);  // all of it is the workgroup's: scalar registers
  s.q0 = __builtin_amdgcn_readfirstlane(s.q0);
  s.len_q = __builtin_amdgcn_readfirstlane(s.len_q);
  s.tile = __builtin_amdgcn_readfirstlane(s.tile);
  s.split_keys = __builtin_amdgcn_readfirstlane(s.split_keys);
  const int tiles = (s.len_q * p.group + rows - 1) / rows;
  if (s.tile < 0 || s.tile >= tiles) {
    s.b = -1;
    return s;
  }
  if (!SORTED || !p.longest_first) s.tile = tiles - 1 - s.tile;  // causal: the rows that see most keys come first
  if (p.kv.table != nullptr) {
    s.k0 = 0;
    s.len_k = paged_keys(p, end_k);
  } else if (p.starts_k != nullptr) {
    s.k0 = clampi(start_k, 0, p.total_k);
    s.len_k = clampi(end_k, s.k0, p.total_k) - s.k0;
  } else {
    s.k0 = 0;
    s.len_k = end_k;
  }
  s.k0 = __builtin_amdgcn_readfirstlane(s.k0);
  s.len_k = __builtin_amdgcn_readfirstlane(s.len_k);
  return s;
}

// Keys that the sequence's row `row`, and all before it, may see end here.
__device__ __forceinline__ int keys_end(const AttnParams& p, const Seq& s, int row) {
  return p.causal ? min(s.len_k, row / p.group + s.len_k - s.len_q + 1) : s.len_k;
}

// What a row's sum is multiplied by, with the weights' sum l: 1 / l, and 0 if the row sees no key (one
// whose scores are all -inf sees keys, and has no largest one: infinity, which makes its zeros NaN).
__device__ __forceinline__ float row_factor(const AttnParams& p, const Seq& s, int row, float l) {
  return keys_end(p, s, row) > 0 ? 1.f / l : 0.f;
}

// The page of key `key` and its place in the page; -1 where the table names no page of the cache.
__device__ __forceinline__ int page_of(const KvSource& kv, const int32_t* table, int key, int& place) {
  const int n = kv.page_shift >= 0 ? key >> kv.page_shift : key / kv.page_size;
  place = key - n * kv.page_size;
  const int page = table[n];
  return (unsigned)page < (unsigned)kv.pages ? page : -1;
}

// Four e4m3 codes (one dword) as four values of T: exact, both types hold every code.
template <typename T>
__device__ __forceinline__ u32x2 e4m3x4(uint32_t c) {
  u32x2 r;
  if constexpr (std::is_same<T, _Float16>::value) {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true));
  } else {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, true));
  }
  return r;
}

// fp16 numbers lose bits below 2^-14 and are zero below 2^-25, so fp16 weights are taken times a power of two
// that puts the largest of a row near the type's end, not at 1: the sums get the same factor and it cancels.
// With it the other keys keep their weights where one key stands far above them (its score 16 above, of 600
// keys: off by 3e-4 of the result, without it by 4e-2).
template <typename T>
constexpr bool kHalf = std::is_same<T, _Float16>::value;

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
// Two floats rounded to nearest even, as one instruction.
template <typename T>
__device__ __forceinline__ uint32_t round2(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef T t2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), t2));
}

// Two floats cut to 16 bits towards zero.
template <typename T>
__device__ __forceinline__ uint32_t cut2(float lo, float hi) {
  if constexpr (kHalf<T>)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
  else
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// What cutting two weights (not negative) to `cut` has left.  Not zero unless the first part is: a value of
// infinity times both is infinity, where 0 or a second part below zero, as rounding leaves, would make it NaN.
// (What is put for zero, the least number of fp16 or the least normal one of bf16, is 2^-39 of the largest
// weight, or less.)
template <typename T>
__device__ __forceinline__ uint32_t rest2(float lo, float hi, uint32_t cut) {
  const float a = lo - from_bits<T>((uint16_t)cut), b = hi - from_bits<T>((uint16_t)(cut >> 16));
  constexpr unsigned short least = kHalf<T> ? 0x0001 : 0x0080;
  const u16x2 some = __builtin_elementwise_min(__builtin_bit_cast(u16x2, cut), u16x2{least, least});
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, round2<T>(a, b)), some));
}

// The larger of two, NaN if one is: two of them are one instruction of three operands, while
// fmaxf takes another to quiet each operand (the row is NaN in the end either way).
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The larger of x in this lane and in lane ^ 32.
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 2^x, the hardware's (relative error about 2^-23; 0 for -infinity).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

typedef u32x4 u32x4_a8 __attribute__((aligned(8)));  // 16 bytes at an address aligned to 8
typedef short s16x4 __attribute__((ext_vector_type(4)));
// Transposing LDS read: the 16 lanes of a group name four rows of 16 consecutive 16-bit
// columns (lane r: row r / 4, columns 4 (r % 4) ..), lane r gets column r of the four rows.
__device__ __forceinline__ u32x2 lds_read_tr(const unsigned char* q) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)q));
}

// ---- values of V that are not finite, at keys that only some rows see ----
// A product adds 0 * v for a masked key, which is NaN where v is infinite or NaN: a row would
// get a value it does not see.  Steps in which some row sees only part of the keys therefore
// look V over first (any_not_finite); in the rare step that holds such a value they are made
// zeros, and when all keys are done a second pass over those steps adds them to the rows that
// see them: kind_ones has 1 where V holds +infinity, -infinity or NaN, and its product with the
// rows' seen keys is positive exactly there.
template <typename T>
constexpr uint32_t kExponents = std::is_same<T, _Float16>::value ? 0x7C007C00u : 0x7F807F80u;

// Whether the stretch of `bytes` of LDS (a multiple of 1024) holds one; the same for all lanes.
template <typename T>
__device__ __forceinline__ bool any_not_finite(const unsigned char* lds, int bytes) {
  u16x2 most = u16x2{0, 0};
  for (int i = 16 * (threadIdx.x & 63); i < bytes; i += 1024) {
    const u32x4 x = *(const u32x4*)(lds + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x[j] & kExponents<T>));
  }
  constexpr unsigned short e = (unsigned short)kExponents<T>;
  return __builtin_amdgcn_ballot_w64(most.x == e || most.y == e) != 0;
}
// kind 0: +infinity, 1: -infinity, 2: NaN
__device__ __forceinline__ float kind_value(int kind) {
  return kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
}
template <typename T>
__device__ __forceinline__ u32x4 kind_ones(u32x4 v, int kind) {
  constexpr uint32_t e = kExponents<T> & 0xFFFF, one = std::is_same<T, _Float16>::value ? 0x3C00u : 0x3F80u;
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r[j] = 0;
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      const uint32_t b = (v[j] >> h) & 0xFFFF;
      const bool hit = kind == 0 ? b == e : kind == 1 ? b == (e | 0x8000) : (b & 0x7FFF) > e;
      r[j] |= hit ? one << h : 0u;
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ u32x4 finite_only(u32x4 v) {
  constexpr uint32_t e = kExponents<T> & 0xFFFF;
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r[j] = ((v[j] & e) == e ? 0u : v[j] & 0xFFFFu) | ((v[j] >> 16 & e) == e ? 0u : v[j] & 0xFFFF0000u);
  return r;
}
// A scale of 8-bit values that is no finite number acts as such values do: it is made zero (in the tile
// kernel in steps that some row sees only part of), and in the second pass the row in LDS gets what its
// codes are with it.
__device__ __forceinline__ bool not_finite(float x) { return !__builtin_isfinite(x); }
template <typename T>
__device__ __forceinline__ u32x4 times(u32x4 v, float scale) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r[j] = round2<T>(from_bits<T>((uint16_t)v[j]) * scale, from_bits<T>((uint16_t)(v[j] >> 16)) * scale);
  return r;
}
// Two 16-bit ones, for keys `key` and `key` + 1 up to `limit`.
template <typename T>
__device__ __forceinline__ uint32_t ones_up_to(int key, int limit) {
  constexpr uint32_t one = std::is_same<T, _Float16>::value ? 0x3C00u : 0x3F80u;
  return (key <= limit ? one : 0u) | (key < limit ? one << 16 : 0u);
}

}  // namespace cmpext3
