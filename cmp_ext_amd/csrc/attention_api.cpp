// C ABI of the attention operators (declared in include/cmpext3_attention.h): checks every
// argument, picks the kernel, tile and split of the keys, and launches on the caller's stream.
#include <hip/hip_runtime_api.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

#include "../../include/cmpext3_attention.h"
#include "attention_params.h"
#include "kernels.h"

using namespace cmpext3;

namespace {

constexpr int kMostDim = 256;  // of a head, in attention and cache
constexpr int64_t kMostThreads = UINT32_MAX;  // of a grid, in one direction
constexpr int kMostHeads = 0xffff;

bool aligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }
bool of8(int64_t a, int64_t b) { return a % 8 == 0 && b % 8 == 0; }

// A cache's sizes, strides and addresses; `paged` also its pages.
int check_cache(const cmpext3_kv_cache& c, bool paged) {
  if (c.kv_dtype != CMPEXT3_F16 && c.kv_dtype != CMPEXT3_BF16 && c.kv_dtype != CMPEXT3_E4M3) return CMPEXT3_ERR_UNSUPPORTED;
  if (c.kv_heads <= 0 || c.dim <= 0) return CMPEXT3_ERR_INVALID_ARG;
  if (c.kv_heads > kMostHeads) return CMPEXT3_ERR_TOO_LARGE;
  if (c.dim % 8 != 0 || c.dim > kMostDim) return CMPEXT3_ERR_UNSUPPORTED;
  // rows of 8 elements: 16 bytes, or 8 of codes
  const size_t row = c.kv_dtype == CMPEXT3_E4M3 ? 8 : 16;
  if (!aligned(c.k, row) || !aligned(c.v, row)) return CMPEXT3_ERR_INVALID_ARG;
  if (!of8(c.k_page, c.v_page) || !of8(c.k_token, c.v_token) || !of8(c.k_head, c.v_head)) return CMPEXT3_ERR_INVALID_ARG;
  if (!paged) return CMPEXT3_OK;
  if (c.pages < 0 || c.page_size <= 0) return CMPEXT3_ERR_INVALID_ARG;
  if (c.pages > 0 && (c.k == nullptr || c.v == nullptr)) return CMPEXT3_ERR_INVALID_ARG;
  if (c.kv_dtype == CMPEXT3_E4M3 && c.pages > 0 && (c.k_scale == nullptr || c.v_scale == nullptr)) return CMPEXT3_ERR_INVALID_ARG;
  return CMPEXT3_OK;
}

void set_source(KvSource& kv, const cmpext3_kv_cache& c) {
  kv.k = c.k;
  kv.v = c.v;
  kv.k_page = c.k_page, kv.k_token = c.k_token, kv.k_head = c.k_head;
  kv.v_page = c.v_page, kv.v_token = c.v_token, kv.v_head = c.v_head;
  kv.k_scale = c.k_scale;
  kv.v_scale = c.v_scale;
  kv.ks_page = c.ks_page, kv.ks_token = c.ks_token, kv.ks_head = c.ks_head;
  kv.vs_page = c.vs_page, kv.vs_token = c.vs_token, kv.vs_head = c.vs_head;
  kv.pages = c.pages;
  kv.page_size = c.page_size;
  kv.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (c.page_size == 1 << i) kv.page_shift = i;
}

struct AttnPlan {
  AttnParams p;
  KvKind kind;
  int hd;        // padded head
  int blocks16;  // few-rows kernel: its tiles of 16 rows; 0: tile kernel
  int waves;     // few-rows kernel: of a workgroup
  int ks;        // tile kernel: groups of waves that share a tile's keys
  int rows;      // of a workgroup
  bool empty;
  int64_t ws_bytes;
};

int plan_attention(const cmpext3_attention_args* a, AttnPlan* out) {
  if (a == nullptr) return CMPEXT3_ERR_INVALID_ARG;
  const cmpext3_kv_cache& c = a->cache;
  const bool paged = a->block_table != nullptr;
  if (a->dtype != CMPEXT3_F16 && a->dtype != CMPEXT3_BF16) return CMPEXT3_ERR_UNSUPPORTED;
  int st = check_cache(c, paged);
  if (st != CMPEXT3_OK) return st;
  if (c.kv_dtype != a->dtype && !(paged && c.kv_dtype == CMPEXT3_E4M3)) return CMPEXT3_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->heads <= 0 || a->heads % c.kv_heads != 0) return CMPEXT3_ERR_INVALID_ARG;
  if (a->heads > kMostHeads) return CMPEXT3_ERR_TOO_LARGE;
  if (!(a->scale > 0.f) || !isfinite(a->scale)) return CMPEXT3_ERR_INVALID_ARG;
  const bool uniform_q = a->starts_q == nullptr;
  if (uniform_q ? a->len_q < 0 : a->total_q < 0) return CMPEXT3_ERR_INVALID_ARG;
  const bool uniform_k = !paged && a->starts_k == nullptr;
  if (!paged && (uniform_k ? a->len_k < 0 : a->total_k < 0)) return CMPEXT3_ERR_INVALID_ARG;
  if (!aligned(a->q, 16) || !aligned(a->out, 8)) return CMPEXT3_ERR_INVALID_ARG;
  if (!of8(a->q_batch, a->q_token) || a->q_head % 8 != 0) return CMPEXT3_ERR_INVALID_ARG;
  if (a->out_batch % 4 != 0 || a->out_token % 4 != 0 || a->out_head % 4 != 0) return CMPEXT3_ERR_INVALID_ARG;

  AttnPlan r{};
  AttnParams& p = r.p;
  const int64_t queries = uniform_q ? (int64_t)a->batch * a->len_q : a->total_q;
  r.empty = queries == 0;
  if (!r.empty && (a->q == nullptr || a->out == nullptr)) return CMPEXT3_ERR_INVALID_ARG;
  if (paged && (a->table_pages < 0 || (a->batch > 0 && a->seq_lens == nullptr))) return CMPEXT3_ERR_INVALID_ARG;
  const int64_t keys = paged ? (int64_t)a->table_pages * c.page_size : uniform_k ? a->len_k : a->total_k;
  if (!paged && keys > 0 && !r.empty && (c.k == nullptr || c.v == nullptr)) return CMPEXT3_ERR_INVALID_ARG;
  const int group = a->heads / c.kv_heads;
  // rows and keys are counted in 32 bits, sums of two numbers of keys too; packed keys addressed
  // within a step in 32
  if (keys > INT_MAX / 2) return CMPEXT3_ERR_TOO_LARGE;
  if (queries > (INT_MAX - 256) / group) return CMPEXT3_ERR_TOO_LARGE;  // their product may pass 64 bits
  if (!paged && (c.k_token < 0 || c.v_token < 0 || std::max(c.k_token, c.v_token) > INT_MAX / (2 * kTileKeys) - kMostDim))
    return CMPEXT3_ERR_TOO_LARGE;

  p.q = a->q;
  p.out = a->out;
  p.q_batch = uniform_q ? a->q_batch : 0, p.q_token = a->q_token, p.q_head = a->q_head;
  p.out_batch = uniform_q ? a->out_batch : 0, p.out_token = a->out_token, p.out_head = a->out_head;
  set_source(p.kv, c);
  if (!paged && !uniform_k) p.kv.k_page = p.kv.v_page = 0;
  p.kv.table = a->block_table;
  p.kv.table_row = a->table_row;
  p.kv.table_pages = a->table_pages;
  p.starts_q = a->starts_q;
  p.starts_k = a->starts_k;
  p.seq_lens = a->seq_lens;
  p.len_q = a->len_q, p.len_k = a->len_k, p.total_q = a->total_q, p.total_k = a->total_k;
  p.batch = a->batch, p.heads = a->heads, p.kv_heads = c.kv_heads, p.group = group, p.dim = c.dim;
  p.causal = a->causal != 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  r.kind = !paged ? kKvPacked : c.kv_dtype == CMPEXT3_E4M3 ? kKvPaged8 : kKvPaged16;
  r.hd = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
  p.splits = 1;
  p.split_keys = INT_MAX;
  if (r.empty) {
    *out = r;
    return CMPEXT3_OK;
  }
  const int64_t mean_rows = queries * group / std::max(a->batch, 1);  // of a sequence and kv head
  r.ks = 1;
  r.blocks16 = paged && mean_rows <= 32 ? (mean_rows <= 16 || r.hd == 256 ? 1 : 2) : 0;
  const int bm = r.rows = r.blocks16 ? 16 * r.blocks16 : 128;
  const int64_t tiles = uniform_q ? (int64_t)a->batch * (((int64_t)a->len_q * group + bm - 1) / bm)
                                  : queries * group / bm + a->batch;
  const int64_t slots = uniform_q ? tiles : tiles + 2;  // and the rows before and behind all sequences
  if (slots * c.kv_heads * 512 > kMostThreads) return CMPEXT3_ERR_TOO_LARGE;
  p.slots = (int)slots;
  // Split the keys where the row tiles alone leave CUs idle.
  const int64_t groups = tiles * c.kv_heads;
  int64_t n = 1;  // splits of the longest sequence
  int least = 0;  // keys of a split at least
  int fit = 0;    // workgroups that splits should fit, found on the device
  if (r.blocks16) {
    // MI355X, one token for each sequence, heads 32 / 8 of 128: two workgroups a CU keep it busy;
    // sequences of one batch differ, so more of them want finer splits to even out (16 of up to
    // 2000 keys: 512 workgroups 20.1 us, 1024 16.0, 2048 20.3; 64 of up to 8192 in 8 bits: splits of 8192
    // keys 153, 2048 130, 1024 124, 512 130), but not below 256 keys, and none where the tiles fill the GPU
    // (64 of up to 1000: 26.1 whole, 31.0 in splits of 512).  A few short ones are latency: 128 keys, one
    // step of each wave (4 of up to 1000 keys: 10.4 us, in splits of 512 14.3).  Over 128 splits joining
    // them costs more than they save (one of 65536, heads 8 / 2: 128 splits 22.2 us, 256 26.9).
    // (`keys` is what the table has room for: with one for 131072 keys splits have 1024, and 64 of up to 8192
    // take 256 us for 189, 4 of up to 4000 21.4 for 15.4.)
    const bool ragged = a->batch > 4;
    least = ragged ? 256 : 128;
    if (groups < 512) n = ((ragged ? 1024 : 512) + groups - 1) / groups;
    n = std::min<int64_t>(std::max<int64_t>(n, keys / 1024), 128);
    // Short keys stay whole where a workgroup is through them sooner than splits are joined (4 of up to 250
    // keys 7.6 and 9.6 in two, 32 of up to 500 11.8 and 15.1, of up to 1000 18.0 and 20.9; but 16 of up to
    // 1000, 128 tiles, 17.1 and 15.4).  Eight waves are through 8-bit keys in half the steps (4 of up to 500
    // keys 8.6 us, 4 waves whole 10.3 and in splits 10.0; 32 of up to 500 9.4, 11.4 and 13.5, of up to 1000
    // 13.9, 18.1 and 16.4; but 4 of up to 1000 11.7, in splits 10.4); of 16-bit keys a CU takes in no more
    // bytes (4 of up to 1000 keys whole: 15.2 with eight waves, when they were tried, 15.9 with four).
    r.waves = 4;
    if (groups <= 256) {
      if (r.kind == kKvPaged8 && r.blocks16 == 1 && r.hd <= 128 && keys > 128 && keys <= (groups >= 128 ? 1024 : 512))
        r.waves = 8, n = 1;
      else if (keys <= 256 || (ragged && keys <= 512) || (groups > 128 && keys <= 1024))
        n = 1;
    }
  } else if (paged) {
    // Two groups of waves share a tile's keys where the tiles do not fill the CUs and the keys are
    // not so long that workgroups of their own pay (16 bits, heads 32 / 8 of 128: 64 new tokens over
    // 8192 keys 43.0 us with one group and 8 splits, 37.4 with two; 16 of up to 64 over up to 4096
    // 50.7 and 42.4; but 4 of up to 512 over up to 8100, 240 tiles, 114 and 129).  (The limits
    // do not take the best everywhere: one of 1024 over 4096, counted as 264 tiles, 90 in two splits, 78 with two groups.)
    // Splits: all at once, two workgroups a CU (8 bits: one of 512 new tokens over 8192 keys, 136 tiles,
    // 255 us whole, 125 in 3, 103 in 4, 125 in 6).  How many keys that is follows from the lengths: up to 62
    // sequences find it on the device (2 of up to 512 over up to 8000 123 us, in 4 splits by the number of
    // tiles 152; 4 of up to 256 over up to 16000 176, in 3 splits 216, in 4 172).  Many uneven tiles even out
    // better in two rounds of splits (30 of up to 60 over up to 3000, 368 tiles, 70.6 and 78.7).
    // Where tiles are many, those that see most keys go first, and no keys are split: 32 of up to 300 new
    // tokens over up to 2000 16-bit keys, 1200 tiles, 118 us in the order of the sequences, 84.5 longest first
    // (60 of up to 100 over 1000, 960 tiles: 68.8 in splits, 41.5; but 60 of up to 60 over up to 4000, 752
    // tiles: 117 in splits, 123).  Packed prompts gained nothing by that order when it was tried (30 of up to
    // 500: 51 us, 63 with it).
    const bool ragged = a->batch > 4;
    least = 256;
    p.longest_first = !uniform_q && ragged && a->batch <= 62 && (groups >= 1024 || (groups >= 512 && keys <= 5 * groups));
    if (p.longest_first) {
      n = 1;
    } else if (r.hd <= 128 && groups <= 256 && (keys <= 4096 || groups <= 32)) {
      r.ks = 2;
      n = std::min<int64_t>(((ragged ? 480 : 256) + groups - 1) / groups, std::max<int64_t>(1, keys / 1024));
    } else if (!uniform_q && a->batch <= 62 && (!ragged || groups <= 256)) {
      fit = 512;
      n = (1536 + groups - 1) / groups;
    } else {
      n = ((ragged ? 1024 : 512) + groups - 1) / groups;
    }
  } else if (groups < 384 && keys >= 512) {
    // Prompts see half their keys, the longest rows first: two groups, or splits, gain where tiles are
    // few and keys long (heads 32 / 8 of 128: one of 1000 tokens, 250 tiles, 25.7 us with one group,
    // 24.6 with two, 33.4 in 2 splits; of 700 19.8 and 20.1, of 300 13.1 and 14.9.  Heads 8 / 2 of 64, one of
    // 2361: 33.1, 27.1 with two groups, 22.1 in 2 splits as well; of 128, one of 4096, 256 tiles: 72.9,
    // 62.5, 58.9 with one group in 3 splits).
    least = 512;
    if (r.hd <= 128 && groups <= (keys >= 2048 ? 160 : 256)) {
      r.ks = 2;
      n = keys >= 2048 ? 2 : 1;
    } else if (keys >= 2048) {
      n = (768 + groups - 1) / groups;
    }
  }
  n = std::min<int64_t>(n, most_splits(bm));
  if (n > 1 && keys > least) {
    const int64_t per = std::max<int64_t>(least, ((keys + n - 1) / n + 127) / 128 * 128);
    const int64_t splits = (keys + per - 1) / per;
    if (splits > 1) {
      p.splits = (int)splits;
      p.split_keys = fit > 0 ? least : (int)per;
      p.fit = fit;
      r.ws_bytes = slots * c.kv_heads * splits * bm * (c.dim + 2) * 4;
    }
  }
  *out = r;
  return CMPEXT3_OK;
}

hipError_t launch_tile_kernel(int dtype, const AttnPlan& r, dim3 grid, hipStream_t s) {
  if (dtype == CMPEXT3_F16) {
    if (r.kind == kKvPacked) return launch_attention_tile_f16_packed(r.hd, r.ks, r.p, grid, s);
    return r.kind == kKvPaged16 ? launch_attention_tile_f16_paged16(r.hd, r.ks, r.p, grid, s) : launch_attention_tile_f16_paged8(r.hd, r.ks, r.p, grid, s);
  }
  if (r.kind == kKvPacked) return launch_attention_tile_bf16_packed(r.hd, r.ks, r.p, grid, s);
  return r.kind == kKvPaged16 ? launch_attention_tile_bf16_paged16(r.hd, r.ks, r.p, grid, s) : launch_attention_tile_bf16_paged8(r.hd, r.ks, r.p, grid, s);
}

hipError_t launch_few_kernel(int dtype, const AttnPlan& r, dim3 grid, hipStream_t s) {
  if (dtype == CMPEXT3_F16)
    return r.kind == kKvPaged16 ? launch_attention_few_f16_paged16(r.hd, r.blocks16, r.waves, r.p, grid, s)
                                : launch_attention_few_f16_paged8(r.hd, r.blocks16, r.waves, r.p, grid, s);
  return r.kind == kKvPaged16 ? launch_attention_few_bf16_paged16(r.hd, r.blocks16, r.waves, r.p, grid, s)
                              : launch_attention_few_bf16_paged8(r.hd, r.blocks16, r.waves, r.p, grid, s);
}

}  // namespace

extern "C" int64_t cmpext3_attention_workspace_size(const cmpext3_attention_args* args) {
  AttnPlan r;
  const int st = plan_attention(args, &r);
  return st != CMPEXT3_OK ? st : r.ws_bytes;
}

extern "C" int cmpext3_attention(const cmpext3_attention_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
  AttnPlan r;
  const int st = plan_attention(args, &r);
  if (st != CMPEXT3_OK || r.empty) return st;
  if (r.ws_bytes > 0) {
    if (workspace == nullptr || workspace_bytes < r.ws_bytes || !aligned(workspace, 16)) return CMPEXT3_ERR_WORKSPACE;
    r.p.part = (float*)workspace;
    r.p.sem = split_counters((hipStream_t)stream, (int64_t)r.p.slots * r.p.kv_heads);
  }
  const dim3 grid((unsigned)((int64_t)r.p.slots * r.p.kv_heads), (unsigned)r.p.splits);
  hipError_t e = r.blocks16 ? launch_few_kernel(args->dtype, r, grid, (hipStream_t)stream)
                            : launch_tile_kernel(args->dtype, r, grid, (hipStream_t)stream);
  if (e == hipSuccess && r.p.splits > 1 && r.p.sem == nullptr)
    e = launch_attention_join(args->dtype, r.rows, r.p, (hipStream_t)stream);
  return (int)e;
}

extern "C" int cmpext3_attention_describe(const cmpext3_attention_args* args, char* buf, int buflen) {
  AttnPlan r;
  const int st = plan_attention(args, &r);
  if (st != CMPEXT3_OK) return st;
  if (buf != nullptr && buflen > 0) {
    static const char* const kinds[] = {"packed", "paged16", "paged8"};
    if (r.empty)
      snprintf(buf, (size_t)buflen, "kernel=none");
    else
      snprintf(buf, (size_t)buflen, "kernel=%s rows=%d groups=%d keys=%s head=%d slots=%d splits=%d split_keys=%d fit=%d%s",
               r.blocks16 ? (r.waves == 8 ? "attention_few8" : "attention_few") : "attention_tile", r.rows, r.ks, kinds[r.kind], r.hd,
               r.p.slots, r.p.splits, r.p.splits > 1 ? r.p.split_keys : 0, r.p.fit, r.p.longest_first ? " order=longest" : "");
  }
  return CMPEXT3_OK;
}

extern "C" int cmpext3_qk_norm_rope(const cmpext3_qk_norm_rope_args* a, void* stream) {
  if (a == nullptr) return CMPEXT3_ERR_INVALID_ARG;
  if (a->dtype != CMPEXT3_F16 && a->dtype != CMPEXT3_BF16 && a->dtype != CMPEXT3_F32) return CMPEXT3_ERR_UNSUPPORTED;
  if (a->heads < 0 || a->kv_heads < 0 || a->tokens < 0 || a->dim <= 0 || a->table_rows < 0) return CMPEXT3_ERR_INVALID_ARG;
  if (a->rotary_dim < 0 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->dim) return CMPEXT3_ERR_INVALID_ARG;
  if (a->dim > 1024) return CMPEXT3_ERR_UNSUPPORTED;
  if (a->heads > kMostHeads || a->kv_heads > kMostHeads) return CMPEXT3_ERR_TOO_LARGE;
  const int64_t per_token = a->heads + a->kv_heads;
  if (a->tokens == 0 || per_token == 0) return CMPEXT3_OK;
  if (a->tokens > kMostThreads / 64 / per_token) return CMPEXT3_ERR_TOO_LARGE;  // a wave per head
  if ((a->heads > 0 && (a->q == nullptr || a->q_out == nullptr)) || (a->kv_heads > 0 && (a->k == nullptr || a->k_out == nullptr)) ||
      a->positions == nullptr || (a->rotary_dim > 0 && a->table_rows > 0 && (a->cos == nullptr || a->sin == nullptr)))
    return CMPEXT3_ERR_INVALID_ARG;
  RopeParams p{};
  p.x[0] = a->q, p.x[1] = a->k;
  p.y[0] = a->q_out, p.y[1] = a->k_out;
  p.x_token[0] = a->q_token, p.x_head[0] = a->q_head, p.x_token[1] = a->k_token, p.x_head[1] = a->k_head;
  p.y_token[0] = a->q_out_token, p.y_head[0] = a->q_out_head, p.y_token[1] = a->k_out_token, p.y_head[1] = a->k_out_head;
  p.weight[0] = a->q_weight, p.weight[1] = a->k_weight;
  p.heads[0] = a->heads, p.heads[1] = a->kv_heads;
  p.dim = a->dim, p.rotary = a->rotary_dim, p.interleaved = a->interleaved != 0;
  p.tokens = a->tokens;
  p.cos = a->cos, p.sin = a->sin;
  p.table_rows = a->table_rows, p.table_row = a->table_row;
  p.positions = a->positions;
  p.eps = a->eps;
  const int per16 = a->dtype == CMPEXT3_F32 ? 4 : 8;  // elements of 16 bytes
  bool vec = a->dim % 16 == 0 && a->rotary_dim % 16 == 0 && a->table_row % 4 == 0 && aligned(a->cos, 16) && aligned(a->sin, 16);
  for (int i = 0; i < 2; ++i)
    vec = vec && aligned(p.x[i], 16) && aligned(p.y[i], 16) && aligned(p.weight[i], 16) && p.x_token[i] % per16 == 0 &&
          p.x_head[i] % per16 == 0 && p.y_token[i] % per16 == 0 && p.y_head[i] % per16 == 0;
  return (int)launch_qk_norm_rope(a->dtype, vec, p, (hipStream_t)stream);
}

namespace {
int cache_params(CacheParams& p, const cmpext3_kv_cache* cache, int dtype, int64_t tokens) {
  if (cache == nullptr || tokens < 0) return CMPEXT3_ERR_INVALID_ARG;
  if (dtype != CMPEXT3_F16 && dtype != CMPEXT3_BF16) return CMPEXT3_ERR_UNSUPPORTED;
  const int st = check_cache(*cache, true);
  if (st != CMPEXT3_OK) return st;
  if (cache->kv_dtype != CMPEXT3_E4M3 && cache->kv_dtype != dtype) return CMPEXT3_ERR_UNSUPPORTED;
  if (tokens > INT_MAX || tokens * cache->kv_heads * 32 > kMostThreads) return CMPEXT3_ERR_TOO_LARGE;  // 32 threads a row at most
  set_source(p.kv, *cache);
  p.kv_heads = cache->kv_heads;
  p.dim = cache->dim;
  p.tokens = tokens;
  return CMPEXT3_OK;
}
}  // namespace

extern "C" int cmpext3_kv_cache_write(const cmpext3_kv_cache* cache, int dtype, const void* k, int64_t k_token, int64_t k_head,
                                      const void* v, int64_t v_token, int64_t v_head, const int64_t* slots, int64_t tokens,
                                      void* stream) {
  CacheParams p{};
  const int st = cache_params(p, cache, dtype, tokens);
  if (st != CMPEXT3_OK) return st;
  if (tokens == 0) return CMPEXT3_OK;
  if (k == nullptr || v == nullptr || slots == nullptr) return CMPEXT3_ERR_INVALID_ARG;
  if (!aligned(k, 16) || !aligned(v, 16) || !of8(k_token, v_token) || !of8(k_head, v_head)) return CMPEXT3_ERR_INVALID_ARG;
  p.k_in = k, p.v_in = v;
  p.k_in_token = k_token, p.k_in_head = k_head, p.v_in_token = v_token, p.v_in_head = v_head;
  p.slots = slots;
  return (int)launch_kv_cache_write(dtype, cache->kv_dtype == CMPEXT3_E4M3, p, (hipStream_t)stream);
}

extern "C" int cmpext3_kv_cache_read(const cmpext3_kv_cache* cache, const int32_t* block_table, int64_t table_row,
                                     int32_t table_pages, const int32_t* starts, int32_t batch, int64_t total, int dtype,
                                     void* k_out, void* v_out, void* stream) {
  CacheParams p{};
  const int st = cache_params(p, cache, dtype, total);
  if (st != CMPEXT3_OK) return st;
  if (batch < 0 || table_pages < 0) return CMPEXT3_ERR_INVALID_ARG;
  if ((int64_t)table_pages * cache->page_size > INT_MAX - kTileKeys) return CMPEXT3_ERR_TOO_LARGE;
  if (total == 0) return CMPEXT3_OK;
  if (k_out == nullptr || v_out == nullptr || (batch > 0 && (starts == nullptr || (table_pages > 0 && block_table == nullptr))))
    return CMPEXT3_ERR_INVALID_ARG;
  if (!aligned(k_out, 16) || !aligned(v_out, 16)) return CMPEXT3_ERR_INVALID_ARG;
  p.kv.table = block_table;
  p.kv.table_row = table_row;
  p.kv.table_pages = table_pages;
  p.starts = starts;
  p.batch = batch;
  p.k_out = k_out, p.v_out = v_out;
  return (int)launch_kv_cache_read(dtype, cache->kv_dtype == CMPEXT3_E4M3, p, (hipStream_t)stream);
}
