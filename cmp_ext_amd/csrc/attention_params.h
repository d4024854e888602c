// Kernel arguments of the attention operators, shared by the host planner and the
// device code.  Strides are in elements.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

namespace cmpext3 {

enum KvKind : int { kKvPacked = 0, kKvPaged16 = 1, kKvPaged8 = 2 };

// Keys per step of the tile kernel, and per step of one wave of the few-rows kernel.
constexpr int kTileKeys = 64;
constexpr int kWaveKeys = 32;

// LDS to join split keys in: a sum for each of 256 threads, a number for each row of a tile and one
// for each of its splits, of which there are so many at most.
constexpr int kJoinBytes = 20 * 1024 + 512;
constexpr int most_splits(int rows_of_tile) { return (kJoinBytes - 4096 - 4 * rows_of_tile) / (4 * rows_of_tile); }

// Keys and values: packed rows, or pages.
struct KvSource {
  const void* k;
  const void* v;
  int64_t k_page, k_token, k_head;  // packed: k_page is the stride between batch entries
  int64_t v_page, v_token, v_head;
  const float* k_scale;  // paged, 8 bits: [pages, page_size, kv_heads]
  const float* v_scale;
  int64_t ks_page, ks_token, ks_head, vs_page, vs_token, vs_head;
  const int32_t* table;  // paged: page numbers, [batch, table_pages]
  int64_t table_row;
  int table_pages, pages, page_size;
  int page_shift;  // log2(page_size), or -1 if that is no power of two
};

struct AttnParams {
  const void* q;
  void* out;
  int64_t q_batch, q_token, q_head, out_batch, out_token, out_head;
  KvSource kv;
  const int32_t* starts_q;  // nullptr: uniform lengths len_q
  const int32_t* starts_k;  // packed keys; nullptr: uniform lengths len_k
  const int32_t* seq_lens;  // paged keys
  int len_q, len_k, total_q, total_k;
  int batch, heads, kv_heads, group, dim;
  int causal;
  float scale_log2;  // scale * log2(e): the softmax runs on powers of two
  int longest_first;  // packed queries, paged keys: row tiles in the order of the keys they see
  int slots;         // row tiles of the grid, for all sequences (see seq_of_slot)
  // split keys: split s of a sequence covers its keys [s * split_keys, (s + 1) * split_keys)
  int splits, split_keys;
  int fit;            // packed queries, paged keys: split_keys is the least, the kernel takes the number of
                      // keys whose splits are at most so many workgroups (fitting_split); 0: it is the number
  float* part;        // sums of the splits (attention_join.h)
  unsigned int* sem;  // counters of the row tiles, or nullptr: joined by a second launch
};

// hd: 64, 128 or 256, the head padded (dim <= hd); ks: groups of waves of a workgroup, each with its
// share of the keys, 1 or (hd up to 128) 2.  grid: slots * kv_heads, splits.
hipError_t launch_attention_tile_f16_packed(int hd, int ks, const AttnParams& p, dim3 grid, hipStream_t s);
hipError_t launch_attention_tile_f16_paged16(int hd, int ks, const AttnParams& p, dim3 grid, hipStream_t s);
hipError_t launch_attention_tile_f16_paged8(int hd, int ks, const AttnParams& p, dim3 grid, hipStream_t s);
hipError_t launch_attention_tile_bf16_packed(int hd, int ks, const AttnParams& p, dim3 grid, hipStream_t s);
hipError_t launch_attention_tile_bf16_paged16(int hd, int ks, const AttnParams& p, dim3 grid, hipStream_t s);
hipError_t launch_attention_tile_bf16_paged8(int hd, int ks, const AttnParams& p, dim3 grid, hipStream_t s);
// blocks16: tiles of 16 rows a workgroup takes, 1 or 2; waves: of a workgroup, 4 or (8 bits,
// one tile, hd up to 128) 8.
hipError_t launch_attention_few_f16_paged16(int hd, int blocks16, int waves, const AttnParams& p, dim3 grid, hipStream_t s);
hipError_t launch_attention_few_f16_paged8(int hd, int blocks16, int waves, const AttnParams& p, dim3 grid, hipStream_t s);
hipError_t launch_attention_few_bf16_paged16(int hd, int blocks16, int waves, const AttnParams& p, dim3 grid, hipStream_t s);
hipError_t launch_attention_few_bf16_paged8(int hd, int blocks16, int waves, const AttnParams& p, dim3 grid, hipStream_t s);
// bm: rows of a row tile.
hipError_t launch_attention_join(int dtype, int bm, const AttnParams& p, hipStream_t s);

struct RopeParams {
  const void* x[2];  // queries, keys
  void* y[2];
  int64_t x_token[2], x_head[2], y_token[2], y_head[2];
  const void* weight[2];
  int heads[2];
  int dim, rotary, interleaved;
  int64_t tokens;
  const float* cos;
  const float* sin;
  int64_t table_rows, table_row;
  const int64_t* positions;
  float eps;
};
// vec: dim and rotary are multiples of 16 and every row of q, k, their outputs and the
// weights is aligned to 16 bytes
hipError_t launch_qk_norm_rope(int dtype, bool vec, const RopeParams& p, hipStream_t s);

struct CacheParams {
  KvSource kv;  // written by the writing kernel
  int kv_heads, dim;
  const void* k_in;
  const void* v_in;
  int64_t k_in_token, k_in_head, v_in_token, v_in_head;
  const int64_t* slots;
  int64_t tokens;  // rows written, or packed rows read
  const int32_t* starts;
  int batch;
  void* k_out;
  void* v_out;
};
hipError_t launch_kv_cache_write(int dtype, bool e4m3, const CacheParams& p, hipStream_t s);
hipError_t launch_kv_cache_read(int dtype, bool e4m3, const CacheParams& p, hipStream_t s);

}  // namespace cmpext3
