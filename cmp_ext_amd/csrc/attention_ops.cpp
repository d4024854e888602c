// Python surface of the attention operators (part of the `_cmpext3` module): tensor checks and
// outputs here, everything else through the C ABI of include/cmpext3_attention.h, on PyTorch's
// current stream of the tensors' device.
#include "attention_ops.h"

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <climits>
#include <cmath>

#include "../../include/cmpext3_attention.h"

namespace {

using OptTensor = c10::optional<torch::Tensor>;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return CMPEXT3_F16;
    case at::kBFloat16: return CMPEXT3_BF16;
    case at::kFloat: return CMPEXT3_F32;
    case at::kFloat8_e4m3fn: return CMPEXT3_E4M3;
    default: return -1;
  }
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void* current_stream(const torch::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

void check_status(int64_t st, const char* op) {
  TORCH_CHECK(st == CMPEXT3_OK, "cmpext3.", op, ": ", cmpext3_status_string((int)st));
}

void check_device(const torch::Tensor& t, const torch::Tensor& like, const char* op, const char* what) {
  TORCH_CHECK(t.is_cuda(), "cmpext3.", op, ": ", what, " must be on a GPU");
  TORCH_CHECK(t.device() == like.device(), "cmpext3.", op, ": device mismatch (", what, ")");
}

// An index tensor the kernels read as a packed vector (or rows, for the block table).
torch::Tensor index_vector(const torch::Tensor& t, at::ScalarType type, int64_t size, const torch::Tensor& like, const char* op,
                           const char* what) {
  TORCH_CHECK(t.dim() == 1, "cmpext3.", op, ": ", what, " must be 1-D");
  TORCH_CHECK(t.scalar_type() == type, "cmpext3.", op, ": ", what, " must be ", c10::toString(type), ", got ", t.scalar_type());
  TORCH_CHECK(t.size(0) == size, "cmpext3.", op, ": ", what, " must have ", size, " elements, got ", t.size(0));
  check_device(t, like, op, what);
  return t.contiguous();
}

// Whether the kernels can read t's heads in place: unit stride inside a head, every other
// stride a multiple of 8 elements, rows of `align` bytes.
bool rows_of_8(const torch::Tensor& t, size_t align) {
  const int64_t d = t.dim() - 1;
  if (t.size(d) > 1 && t.stride(d) != 1) return false;
  for (int64_t i = 0; i < d; ++i)
    if (t.size(i) > 1 && (t.stride(i) % 8 != 0 || t.stride(i) < 0)) return false;
  return t.numel() == 0 || (uintptr_t)t.data_ptr() % align == 0;
}
// t itself, or a packed copy the kernels can read.
torch::Tensor readable(const torch::Tensor& t) {
  if (rows_of_8(t, 16)) return t;
  torch::Tensor c = torch::empty(t.sizes(), t.options());
  c.copy_(t);
  return c;
}
// The stride of dimension i, 0 where it is never used.
int64_t step_of(const torch::Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; }

int checked_int(int64_t v, const char* op, const char* what) {
  TORCH_CHECK(v <= INT_MAX, "cmpext3.", op, ": ", what, " = ", v, " exceeds the supported range (2^31 - 1)");
  return (int)v;
}

void check_head(int64_t dim, const char* op) {
  TORCH_CHECK(dim > 0 && dim % 8 == 0 && dim <= 256, "cmpext3.", op, ": the head size must be a multiple of 8 up to 256, got ", dim);
}

// The caches and their scales, checked against each other.
cmpext3_kv_cache cache_of(const torch::Tensor& k, const torch::Tensor& v, const OptTensor& ks, const OptTensor& vs, const char* op) {
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4, "cmpext3.", op, ": the caches must be [pages, page_size, kv_heads, dim]");
  TORCH_CHECK(k.sizes() == v.sizes(), "cmpext3.", op, ": cache shape mismatch ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), "cmpext3.", op, ": cache dtype mismatch");
  const bool e4m3 = k.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(e4m3 || k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16, "cmpext3.", op,
              ": unsupported cache dtype ", k.scalar_type(), " (float16, bfloat16 or float8_e4m3fn)");
  TORCH_CHECK(k.size(1) > 0 && k.size(2) > 0, "cmpext3.", op, ": empty pages or no heads");
  check_head(k.size(3), op);
  TORCH_CHECK(given(ks) == e4m3 && given(vs) == e4m3, "cmpext3.", op, e4m3 ? ": a float8_e4m3fn cache needs k_scale and v_scale"
                                                                        : ": only a float8_e4m3fn cache has scales");
  TORCH_CHECK(rows_of_8(k, e4m3 ? 8 : 16) && rows_of_8(v, e4m3 ? 8 : 16), "cmpext3.", op,
              ": the caches need unit stride inside a head, other strides of multiples of 8 elements and aligned rows");
  cmpext3_kv_cache c{};
  c.kv_dtype = dtype_code(k.scalar_type());
  c.pages = checked_int(k.size(0), op, "pages");
  c.page_size = checked_int(k.size(1), op, "page_size");
  c.kv_heads = checked_int(k.size(2), op, "kv_heads");
  c.dim = (int)k.size(3);
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.k_page = step_of(k, 0), c.k_token = step_of(k, 1), c.k_head = step_of(k, 2);
  c.v_page = step_of(v, 0), c.v_token = step_of(v, 1), c.v_head = step_of(v, 2);
  if (e4m3) {
    for (const torch::Tensor* s : {&*ks, &*vs}) {
      TORCH_CHECK(s->scalar_type() == at::kFloat && s->dim() == 3 && s->sizes() == k.sizes().slice(0, 3), "cmpext3.", op,
                  ": the scales must be float32 [pages, page_size, kv_heads]");
    }
    c.k_scale = (float*)ks->data_ptr();
    c.v_scale = (float*)vs->data_ptr();
    c.ks_page = step_of(*ks, 0), c.ks_token = step_of(*ks, 1), c.ks_head = step_of(*ks, 2);
    c.vs_page = step_of(*vs, 0), c.vs_token = step_of(*vs, 1), c.vs_head = step_of(*vs, 2);
  }
  return c;
}

void check_cache_device(const torch::Tensor& k, const torch::Tensor& v, const OptTensor& ks, const OptTensor& vs, const torch::Tensor& like,
                        const char* op) {
  check_device(k, like, op, "k_cache");
  check_device(v, like, op, "v_cache");
  if (given(ks)) check_device(*ks, like, op, "k_scale");
  if (given(vs)) check_device(*vs, like, op, "v_scale");
}

torch::Tensor table_of(const torch::Tensor& t, const torch::Tensor& like, const char* op) {
  TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kInt, "cmpext3.", op, ": block_table must be int32 [batch, pages]");
  check_device(t, like, op, "block_table");
  return t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t;
}

void run_attention(cmpext3_attention_args& a, const torch::Tensor& like, const char* op) {
  const int64_t need = cmpext3_attention_workspace_size(&a);
  check_status(need < 0 ? need : CMPEXT3_OK, op);
  torch::Tensor ws;
  if (need > 0) ws = torch::empty({need}, like.options().dtype(torch::kUInt8));
  check_status(cmpext3_attention(&a, ws.defined() ? ws.data_ptr() : nullptr, need, current_stream(like)), op);
}

float scale_of(c10::optional<double> scale, int64_t dim, const char* op) {
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt((double)dim);
  TORCH_CHECK(s > 0 && std::isfinite((float)s) && (float)s > 0, "cmpext3.", op, ": scale must be positive and finite, got ", s);
  return (float)s;
}

// qk_norm_rope(q[tokens, heads, dim], k[tokens, kv_heads, dim], cos, sin, positions, ...)
std::tuple<torch::Tensor, torch::Tensor> qk_norm_rope(const torch::Tensor& q_in, const torch::Tensor& k_in, const torch::Tensor& cos,
                                                      const torch::Tensor& sin, const torch::Tensor& positions,
                                                      const OptTensor& q_weight, const OptTensor& k_weight, double eps,
                                                      bool interleaved) {
  const char* op = "qk_norm_rope";
  TORCH_CHECK(q_in.dim() == 3 && k_in.dim() == 3, "cmpext3.", op, ": q and k must be [tokens, heads, dim]");
  TORCH_CHECK(q_in.scalar_type() == k_in.scalar_type(), "cmpext3.", op, ": dtype mismatch");
  const int code = dtype_code(q_in.scalar_type());
  TORCH_CHECK(code == CMPEXT3_F16 || code == CMPEXT3_BF16 || code == CMPEXT3_F32, "cmpext3.", op, ": unsupported dtype ", q_in.scalar_type());
  const int64_t tokens = q_in.size(0), dim = q_in.size(2);
  TORCH_CHECK(k_in.size(0) == tokens && k_in.size(2) == dim, "cmpext3.", op, ": shape mismatch ", q_in.sizes(), " and ", k_in.sizes());
  TORCH_CHECK(dim > 0 && dim <= 1024, "cmpext3.", op, ": the head size must be 1 to 1024, got ", dim);
  TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat,
              "cmpext3.", op, ": cos and sin must be float32 [positions, rotary_dim / 2]");
  TORCH_CHECK(2 * cos.size(1) <= dim, "cmpext3.", op, ": the tables turn ", 2 * cos.size(1), " elements of a head of ", dim);
  TORCH_CHECK(eps >= 0 && std::isfinite(eps), "cmpext3.", op, ": eps must be finite and not negative");
  check_device(q_in, q_in, op, "q");
  check_device(k_in, q_in, op, "k");
  check_device(cos, q_in, op, "cos");
  check_device(sin, q_in, op, "sin");
  c10::DeviceGuard guard(q_in.device());
  const torch::Tensor pos = index_vector(positions, at::kLong, tokens, q_in, op, "positions");
  // heads of unit stride are read in place, whatever the other strides
  const torch::Tensor q = dim > 1 && q_in.stride(2) != 1 ? q_in.contiguous() : q_in;
  const torch::Tensor k = dim > 1 && k_in.stride(2) != 1 ? k_in.contiguous() : k_in;
  torch::Tensor c = cos.contiguous(), s = sin.contiguous();
  torch::Tensor w[2];
  const OptTensor* given_w[2] = {&q_weight, &k_weight};
  for (int i = 0; i < 2; ++i) {
    if (!given(*given_w[i])) continue;
    w[i] = **given_w[i];
    TORCH_CHECK(w[i].dim() == 1 && w[i].size(0) == dim && w[i].scalar_type() == q.scalar_type(), "cmpext3.", op,
                ": weights must be [dim] of the dtype of q and k");
    check_device(w[i], q, op, "weights");
    w[i] = w[i].contiguous();
  }
  torch::Tensor qo = torch::empty(q.sizes(), q.options()), ko = torch::empty(k.sizes(), k.options());
  cmpext3_qk_norm_rope_args a{};
  a.dtype = code;
  a.interleaved = interleaved;
  a.heads = checked_int(q.size(1), op, "heads");
  a.kv_heads = checked_int(k.size(1), op, "kv_heads");
  a.dim = (int)dim;
  a.rotary_dim = (int)(2 * c.size(1));
  a.tokens = tokens;
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.q_out = qo.data_ptr(), a.k_out = ko.data_ptr();
  a.q_token = step_of(q, 0), a.q_head = step_of(q, 1), a.k_token = step_of(k, 0), a.k_head = step_of(k, 1);
  a.q_out_token = step_of(qo, 0), a.q_out_head = step_of(qo, 1), a.k_out_token = step_of(ko, 0), a.k_out_head = step_of(ko, 1);
  a.q_weight = w[0].defined() ? w[0].data_ptr() : nullptr;
  a.k_weight = w[1].defined() ? w[1].data_ptr() : nullptr;
  a.cos = (const float*)c.data_ptr(), a.sin = (const float*)s.data_ptr();
  a.table_rows = c.size(0), a.table_row = c.size(1);
  a.positions = (const int64_t*)pos.data_ptr();
  a.eps = (float)eps;
  check_status(cmpext3_qk_norm_rope(&a, current_stream(q)), op);
  return {qo, ko};
}

void kv_cache_write(const torch::Tensor& k_in, const torch::Tensor& v_in, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                    const torch::Tensor& slots, const OptTensor& k_scale, const OptTensor& v_scale) {
  const char* op = "kv_cache_write";
  const cmpext3_kv_cache c = cache_of(k_cache, v_cache, k_scale, v_scale, op);
  TORCH_CHECK(k_in.dim() == 3 && k_in.sizes() == v_in.sizes() && k_in.size(1) == c.kv_heads && k_in.size(2) == c.dim, "cmpext3.", op,
              ": k and v must be [tokens, kv_heads, dim] like the cache, got ", k_in.sizes(), " and ", v_in.sizes());
  const int code = dtype_code(k_in.scalar_type());
  TORCH_CHECK((code == CMPEXT3_F16 || code == CMPEXT3_BF16) && k_in.scalar_type() == v_in.scalar_type(), "cmpext3.", op,
              ": k and v must be float16 or bfloat16");
  TORCH_CHECK(c.kv_dtype == CMPEXT3_E4M3 || c.kv_dtype == code, "cmpext3.", op, ": dtype mismatch with the cache");
  check_cache_device(k_cache, v_cache, k_scale, v_scale, k_cache, op);
  check_device(k_in, k_cache, op, "k");
  check_device(v_in, k_cache, op, "v");
  c10::DeviceGuard guard(k_cache.device());
  const torch::Tensor at = index_vector(slots, at::kLong, k_in.size(0), k_cache, op, "slots");
  const torch::Tensor k = readable(k_in), v = readable(v_in);
  check_status(cmpext3_kv_cache_write(&c, code, k.data_ptr(), step_of(k, 0), step_of(k, 1), v.data_ptr(), step_of(v, 0), step_of(v, 1),
                                      (const int64_t*)at.data_ptr(), k.size(0), current_stream(k_cache)),
               op);
}

std::tuple<torch::Tensor, torch::Tensor> kv_cache_read(const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                                                       const torch::Tensor& block_table, const torch::Tensor& cu_seqlens, int64_t total,
                                                       c10::optional<at::ScalarType> dtype, const OptTensor& k_scale,
                                                       const OptTensor& v_scale) {
  const char* op = "kv_cache_read";
  const cmpext3_kv_cache c = cache_of(k_cache, v_cache, k_scale, v_scale, op);
  const at::ScalarType type = dtype.has_value() ? *dtype : k_cache.scalar_type();
  const int code = dtype_code(type);
  TORCH_CHECK(code == CMPEXT3_F16 || code == CMPEXT3_BF16, "cmpext3.", op, ": dtype must be float16 or bfloat16");
  TORCH_CHECK(c.kv_dtype == CMPEXT3_E4M3 || c.kv_dtype == code, "cmpext3.", op, ": dtype mismatch with the cache");
  TORCH_CHECK(total >= 0, "cmpext3.", op, ": total must not be negative");
  check_cache_device(k_cache, v_cache, k_scale, v_scale, k_cache, op);
  c10::DeviceGuard guard(k_cache.device());
  const torch::Tensor table = table_of(block_table, k_cache, op);
  const int64_t batch = table.size(0);
  const torch::Tensor starts = index_vector(cu_seqlens, at::kInt, batch + 1, k_cache, op, "cu_seqlens");
  const auto options = k_cache.options().dtype(type);
  torch::Tensor k = torch::empty({total, c.kv_heads, c.dim}, options), v = torch::empty({total, c.kv_heads, c.dim}, options);
  check_status(cmpext3_kv_cache_read(&c, (const int32_t*)table.data_ptr(), step_of(table, 0), checked_int(table.size(1), op, "table pages"),
                                     (const int32_t*)starts.data_ptr(), checked_int(batch, op, "batch"), total, code, k.data_ptr(),
                                     v.data_ptr(), current_stream(k_cache)),
               op);
  return {k, v};
}

// attention: [batch, tokens, heads, dim] of uniform lengths, or packed [tokens, heads, dim]
torch::Tensor attention(const torch::Tensor& q_in, const torch::Tensor& k_in, const torch::Tensor& v_in, const OptTensor& cu_q,
                        const OptTensor& cu_k, bool causal, c10::optional<double> scale) {
  const char* op = "attention";
  const int64_t nd = q_in.dim();
  TORCH_CHECK((nd == 3 || nd == 4) && k_in.dim() == nd && v_in.dim() == nd, "cmpext3.", op,
              ": q, k and v must be [tokens, heads, dim] or [batch, tokens, heads, dim]");
  TORCH_CHECK(k_in.sizes() == v_in.sizes(), "cmpext3.", op, ": shape mismatch ", k_in.sizes(), " and ", v_in.sizes());
  const int64_t heads = q_in.size(nd - 2), kv_heads = k_in.size(nd - 2), dim = q_in.size(nd - 1);
  TORCH_CHECK(k_in.size(nd - 1) == dim, "cmpext3.", op, ": head size mismatch");
  TORCH_CHECK(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "cmpext3.", op, ": ", heads, " heads are no multiple of ", kv_heads);
  const int code = dtype_code(q_in.scalar_type());
  TORCH_CHECK(code == CMPEXT3_F16 || code == CMPEXT3_BF16, "cmpext3.", op, ": unsupported dtype ", q_in.scalar_type());
  TORCH_CHECK(k_in.scalar_type() == q_in.scalar_type() && v_in.scalar_type() == q_in.scalar_type(), "cmpext3.", op, ": dtype mismatch");
  check_head(dim, op);
  TORCH_CHECK(given(cu_q) == given(cu_k), "cmpext3.", op, ": cu_seqlens_q and cu_seqlens_k go together");
  TORCH_CHECK(!given(cu_q) || nd == 3, "cmpext3.", op, ": cu_seqlens need packed [tokens, heads, dim]");
  TORCH_CHECK(nd == 3 || k_in.size(0) == q_in.size(0), "cmpext3.", op, ": batch size mismatch");
  cmpext3_attention_args a{};
  a.scale = scale_of(scale, dim, op);
  check_device(q_in, q_in, op, "q");
  check_device(k_in, q_in, op, "k");
  check_device(v_in, q_in, op, "v");
  c10::DeviceGuard guard(q_in.device());
  const torch::Tensor q = readable(q_in), k = readable(k_in), v = readable(v_in);
  torch::Tensor out = torch::empty(q.sizes(), q.options()), starts_q, starts_k;
  a.dtype = code;
  a.heads = checked_int(heads, op, "heads");
  a.causal = causal;
  const int64_t t = nd - 3;  // the token dimension
  const int tq = checked_int(q.size(t), op, "tokens"), tk = checked_int(k.size(t), op, "tokens");
  if (given(cu_q)) {
    TORCH_CHECK(cu_q->dim() == 1 && cu_q->size(0) >= 1, "cmpext3.", op, ": cu_seqlens_q must be 1-D, one more than the sequences");
    a.batch = checked_int(cu_q->size(0) - 1, op, "batch");
    starts_q = index_vector(*cu_q, at::kInt, a.batch + 1, q, op, "cu_seqlens_q");
    starts_k = index_vector(*cu_k, at::kInt, a.batch + 1, q, op, "cu_seqlens_k");
    a.starts_q = (const int32_t*)starts_q.data_ptr();
    a.starts_k = (const int32_t*)starts_k.data_ptr();
    a.total_q = tq, a.total_k = tk;
  } else {
    a.batch = nd == 4 ? checked_int(q.size(0), op, "batch") : 1;
    a.len_q = tq, a.len_k = tk;
  }
  a.q = q.data_ptr(), a.out = out.data_ptr();
  a.q_token = step_of(q, t), a.q_head = step_of(q, t + 1), a.out_token = step_of(out, t), a.out_head = step_of(out, t + 1);
  a.cache.kv_dtype = code;
  a.cache.kv_heads = checked_int(kv_heads, op, "kv_heads");
  a.cache.dim = (int)dim;
  a.cache.k = k.data_ptr(), a.cache.v = v.data_ptr();
  a.cache.k_token = step_of(k, t), a.cache.k_head = step_of(k, t + 1);
  a.cache.v_token = step_of(v, t), a.cache.v_head = step_of(v, t + 1);
  if (nd == 4) {
    a.q_batch = step_of(q, 0), a.out_batch = step_of(out, 0);
    a.cache.k_page = step_of(k, 0), a.cache.v_page = step_of(v, 0);
  }
  run_attention(a, q, op);
  return out;
}

torch::Tensor paged_attention(const torch::Tensor& q_in, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                              const torch::Tensor& block_table, const torch::Tensor& seq_lens, const OptTensor& cu_q,
                              const OptTensor& k_scale, const OptTensor& v_scale, bool causal, c10::optional<double> scale) {
  const char* op = "paged_attention";
  cmpext3_attention_args a{};
  a.cache = cache_of(k_cache, v_cache, k_scale, v_scale, op);
  TORCH_CHECK(q_in.dim() == 3, "cmpext3.", op, ": q must be [tokens, heads, dim]");
  const int64_t heads = q_in.size(1);
  TORCH_CHECK(q_in.size(2) == a.cache.dim, "cmpext3.", op, ": head size mismatch with the cache");
  TORCH_CHECK(heads > 0 && heads % a.cache.kv_heads == 0, "cmpext3.", op, ": ", heads, " heads are no multiple of ", a.cache.kv_heads);
  const int code = dtype_code(q_in.scalar_type());
  TORCH_CHECK(code == CMPEXT3_F16 || code == CMPEXT3_BF16, "cmpext3.", op, ": unsupported dtype ", q_in.scalar_type());
  TORCH_CHECK(a.cache.kv_dtype == CMPEXT3_E4M3 || a.cache.kv_dtype == code, "cmpext3.", op, ": dtype mismatch with the cache");
  a.scale = scale_of(scale, a.cache.dim, op);
  check_device(q_in, q_in, op, "q");
  check_cache_device(k_cache, v_cache, k_scale, v_scale, q_in, op);
  c10::DeviceGuard guard(q_in.device());
  const torch::Tensor table = table_of(block_table, q_in, op);
  const int64_t batch = table.size(0);
  const torch::Tensor lens = index_vector(seq_lens, at::kInt, batch, q_in, op, "seq_lens");
  const torch::Tensor q = readable(q_in);
  torch::Tensor out = torch::empty(q.sizes(), q.options()), starts;
  a.dtype = code;
  a.batch = checked_int(batch, op, "batch");
  a.heads = checked_int(heads, op, "heads");
  a.causal = causal;
  if (given(cu_q)) {
    starts = index_vector(*cu_q, at::kInt, batch + 1, q, op, "cu_seqlens_q");
    if (batch == 0) return out.zero_();
    a.starts_q = (const int32_t*)starts.data_ptr();
    a.total_q = checked_int(q.size(0), op, "tokens");
  } else {
    TORCH_CHECK(q.size(0) == batch, "cmpext3.", op, ": without cu_seqlens_q there is one token for each of the ", batch,
                " sequences, got ", q.size(0));
    a.len_q = 1;
  }
  a.q = q.data_ptr(), a.out = out.data_ptr();
  a.q_token = step_of(q, 0), a.q_head = step_of(q, 1), a.out_token = step_of(out, 0), a.out_head = step_of(out, 1);
  a.q_batch = a.q_token, a.out_batch = a.out_token;
  a.block_table = (const int32_t*)table.data_ptr();
  a.table_row = step_of(table, 0);
  a.table_pages = checked_int(table.size(1), op, "table pages");
  a.seq_lens = (const int32_t*)lens.data_ptr();
  if (a.table_pages == 0 || batch == 0) return out.zero_();  // no keys at all
  run_attention(a, q, op);
  return out;
}

}  // namespace

void register_attention_ops(py::module& m) {
  m.def("qk_norm_rope", &qk_norm_rope, "Norms of queries and keys for each head with the position rotation, in one pass",
        py::arg("q"), py::arg("k"), py::arg("cos"), py::arg("sin"), py::arg("positions"), py::arg("q_weight") = py::none(),
        py::arg("k_weight") = py::none(), py::arg("eps") = 1e-6, py::arg("interleaved") = false);
  m.def("kv_cache_write", &kv_cache_write, "Write keys and values into a paged cache (16 bits, or 8 with scales)", py::arg("k"),
        py::arg("v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"), py::arg("k_scale") = py::none(),
        py::arg("v_scale") = py::none());
  m.def("kv_cache_read", &kv_cache_read, "Read sequences of a paged cache back as packed rows", py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("cu_seqlens"), py::arg("total"), py::arg("dtype") = py::none(), py::arg("k_scale") = py::none(),
        py::arg("v_scale") = py::none());
  m.def("attention", &attention, "softmax(scale q k^T) v over packed or batched prompts, with grouped heads", py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("cu_seqlens_q") = py::none(), py::arg("cu_seqlens_k") = py::none(), py::arg("causal") = true,
        py::arg("scale") = py::none());
  m.def("paged_attention", &paged_attention, "Attention of new tokens over a paged cache (16 bits, or 8 with scales)", py::arg("q"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"), py::arg("seq_lens"), py::arg("cu_seqlens_q") = py::none(),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(), py::arg("causal") = true, py::arg("scale") = py::none());
}
