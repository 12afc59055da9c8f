// paged.cpp — the paged-cache operators of the C++ host API (see mlxq.hpp): shape checks, workspaces and the calls of
// the C ABI.
#include <cmath>

#include "../../include/mlxq.h"
#include "mlxq.hpp"

namespace mlxq {

namespace {

void check(int status) {
  if (status != MLXQ_OK) throw Error(status, mlxq_last_error());
}
[[noreturn]] void bad(const std::string& msg) { throw Error(MLXQ_EINVAL, msg); }

int abi_dtype(Dtype dt, const char* op) {
  if (dt == Dtype::Float32) return MLXQ_FLOAT32;
  if (dt == Dtype::Bfloat16) return MLXQ_BFLOAT16;
  if (dt == Dtype::Float16) return MLXQ_FLOAT16;
  bad(std::string(op) + ": expected a float32, bfloat16 or float16 array, got " + dtype_name(dt));
}

mlxq_heads heads_of(const Array& x, const char* op, const char* what) {
  if (x.ndim() != 3) bad(std::string(op) + ": " + what + " must be [tokens, heads, head_dim]");
  return {x.data(), x.dim(1), x.dim(1) * x.dim(2), x.dim(2)};
}

const int32_t* ints(const Array& a, std::vector<int64_t> shape, const char* op, const char* what) {
  if (a.dtype() != Dtype::Int32 || a.shape() != shape) bad(std::string(op) + ": " + what + " has another shape or is not int32");
  return (const int32_t*)a.data();
}
const float* floats(const std::optional<Array>& a, int64_t n, const char* op, const char* what) {
  if (!a) return nullptr;
  if (a->dtype() != Dtype::Float32 || a->shape() != std::vector<int64_t>{n})
    bad(std::string(op) + ": " + what + " must be float32 of one value a query head");
  return (const float*)a->data();
}

mlxq_paged_cache cache_of(const Array& k, const Array& v, const char* op) {
  const int dt = abi_dtype(k.dtype(), op);
  const int64_t C = 16 / (int64_t)dtype_size(k.dtype());
  if (k.ndim() != 6 || v.ndim() != 5 || k.dim(4) != 16 || k.dim(5) != C)
    bad(std::string(op) + ": k_cache must be [pages, heads, page_size/16, head_dim/C, 16, C], v_cache [pages, heads, page_size/C, head_dim, C]");
  const int64_t pages = k.dim(0), heads = k.dim(1), P = k.dim(2) * 16, D = k.dim(3) * C;
  if (v.dtype() != k.dtype() || v.shape() != std::vector<int64_t>{pages, heads, P / C, D, C})
    bad(std::string(op) + ": v_cache does not match k_cache");
  return {k.data(), v.data(), heads * P * D, heads * P * D, pages, P, heads, D, dt};
}

mlxq_paged_batch batch_of(const CacheBatch& b, const char* op) {
  if (b.block_tables.ndim() != 2) bad(std::string(op) + ": block_tables must be 2-D");
  const int64_t B = b.block_tables.dim(0), width = b.block_tables.dim(1);
  mlxq_paged_batch r = {};
  r.block_tables = ints(b.block_tables, {B, width}, op, "block_tables");
  r.q_starts = ints(b.q_starts, {B + 1}, op, "q_starts");
  r.kv_lens = ints(b.kv_lens, {B}, op, "kv_lens");
  r.sequences = B;
  r.table_width = r.table_stride = width;
  r.max_q = b.max_q;
  r.max_kv = b.max_kv;
  return r;
}

void table_of(const Array& t, const char* op, const float*& p, int64_t& rows, int64_t& R) {
  if (t.ndim() != 3 || t.dim(2) != 2 || t.dtype() != Dtype::Float32)
    bad(std::string(op) + ": table must be float32 [positions, rotary_dim/2, 2]");
  p = (const float*)t.data();
  rows = t.dim(0);
  R = 2 * t.dim(1);
}

}  // namespace

RotaryFrequencies rotary_frequencies(int64_t rotary_dim, double base, int kind, double factor, double original_context,
                                     double low, double high) {
  const mlxq_rope_scaling s = {kind, factor, original_context, low, high};
  RotaryFrequencies f;
  f.inv_freq.resize(rotary_dim > 0 && rotary_dim <= 256 ? rotary_dim / 2 : 0);
  check(mlxq_rotary_frequencies(rotary_dim, base, &s, f.inv_freq.data(), &f.magnitude));
  return f;
}

Array rotary_table(int64_t positions, const RotaryFrequencies& f, hipStream_t s) {
  Array t = Array::empty({positions, (int64_t)f.inv_freq.size(), 2}, Dtype::Float32);
  check(mlxq_rotary_table(f.inv_freq.data(), 2 * (int64_t)f.inv_freq.size(), f.magnitude, positions, (float*)t.data(), s));
  return t;
}

Array rotary(const Array& x, const Array& positions, const Array& table, bool interleaved, bool inverse, hipStream_t s) {
  const char* op = "rotary";
  const int dt = abi_dtype(x.dtype(), op);
  const mlxq_heads xh = heads_of(x, op, "x");
  const float* t;
  int64_t rows, R;
  table_of(table, op, t, rows, R);
  const int32_t* pos = ints(positions, {x.dim(0)}, op, "positions");
  Array y = Array::empty(x.shape(), x.dtype());
  const mlxq_heads yh = heads_of(y, op, "y");
  check(mlxq_rotary(&xh, dt, x.dim(0), x.dim(2), pos, t, rows, R, interleaved, inverse, &yh, s));
  return y;
}

std::pair<std::vector<int64_t>, std::vector<int64_t>> cache_shapes(int64_t pages, int64_t heads, int64_t page_size,
                                                                   int64_t head_dim, Dtype dt) {
  const int64_t C = 16 / (int64_t)dtype_size(dt);
  return {{pages, heads, page_size / 16, head_dim / C, 16, C}, {pages, heads, page_size / C, head_dim, C}};
}

Array cache_append(const Array& k, const Array& v, const Array& k_cache, const Array& v_cache, const CacheBatch& batch,
                   const Array* q, const Array* table, const Array* positions, bool interleaved, hipStream_t s) {
  const char* op = "cache_append";
  const mlxq_paged_cache c = cache_of(k_cache, v_cache, op);
  const mlxq_paged_batch b = batch_of(batch, op);
  const mlxq_heads kh = heads_of(k, op, "k"), vh = heads_of(v, op, "v");
  const int64_t T = k.dim(0);
  const std::vector<int64_t> shape = {T, c.heads, c.head_dim};
  if (k.shape() != shape || v.shape() != shape || k.dtype() != k_cache.dtype() || v.dtype() != k_cache.dtype())
    bad("cache_append: k and v must be [tokens, heads, head_dim] of the cache's heads and dtype");
  const float* t = nullptr;
  int64_t rows = 0, R = 0;
  if (table) table_of(*table, op, t, rows, R);
  const int32_t* pos = positions ? ints(*positions, {T}, op, "positions") : nullptr;
  Array out;
  mlxq_heads qh = {}, oh = {};
  if (q) {
    qh = heads_of(*q, op, "q");
    if (q->dim(0) != T || q->dim(2) != c.head_dim || q->dtype() != k_cache.dtype())
      bad("cache_append: q does not fit the step or the cache");
    out = Array::empty(q->shape(), q->dtype());
    oh = heads_of(out, op, "q_out");
  }
  check(mlxq_cache_append(&kh, &vh, T, &c, &b, pos, t, rows, R, interleaved, q ? &qh : nullptr, q ? &oh : nullptr, s));
  return out;
}

void PagedAttention::forward_into(const Array& q, const Array& k_cache, const Array& v_cache, const CacheBatch& batch,
                                  const Array& out, hipStream_t s) const {
  const char* op = "paged_attention";
  const mlxq_paged_cache c = cache_of(k_cache, v_cache, op);
  const mlxq_paged_batch b = batch_of(batch, op);
  const mlxq_heads qh = heads_of(q, op, "q"), oh = heads_of(out, op, "out");
  if (q.dim(2) != c.head_dim || q.dtype() != k_cache.dtype()) bad("paged_attention: q does not fit the cache");
  if (out.shape() != q.shape() || out.dtype() != q.dtype()) bad("paged_attention: out must have q's shape and dtype");
  mlxq_attention o = {};
  o.scale = scale != 0.0f ? scale : (float)(1.0 / std::sqrt((double)c.head_dim));
  o.causal = causal;
  o.window = window;
  o.softcap = softcap;
  o.prefix_lens = prefix_lens ? ints(*prefix_lens, {b.sequences}, op, "prefix_lens") : nullptr;
  o.alibi_slopes = floats(alibi_slopes, q.dim(1), op, "alibi_slopes");
  o.sinks = floats(sinks, q.dim(1), op, "sinks");
  const size_t need = mlxq_paged_attention_workspace_size(q.dim(0), q.dim(1), &c, &b, &o);
  const Array& ws = workspace_.at_least(need);
  check(mlxq_paged_attention(&qh, q.dim(0), &c, &b, &o, &oh, ws.data(), ws.nbytes(), s));
}

Array PagedAttention::forward(const Array& q, const Array& k_cache, const Array& v_cache, const CacheBatch& batch,
                              hipStream_t s) const {
  Array out = Array::empty(q.shape(), q.dtype());
  forward_into(q, k_cache, v_cache, batch, out, s);
  return out;
}

void copy_pages(const Array& cache, int dim, const Array& src, const Array& dst, const Array* block_tables, hipStream_t s) {
  if (dim < 0 || dim >= cache.ndim() - 1) bad("copy_pages: no dimension of pages");
  if (src.ndim() != 1) bad("copy_pages: src must be 1-D");
  int64_t planes = 1, page = (int64_t)dtype_size(cache.dtype());
  for (int i = 0; i < dim; ++i) planes *= cache.dim(i);
  for (int i = dim + 1; i < cache.ndim(); ++i) page *= cache.dim(i);
  const int64_t n = src.dim(0), pages = cache.dim(dim);
  int32_t* t = nullptr;
  int64_t rows = 0, width = 0;
  if (block_tables) {
    if (block_tables->ndim() != 2) bad("copy_pages: block_tables must be 2-D");
    rows = block_tables->dim(0);
    width = block_tables->dim(1);
    t = const_cast<int32_t*>(ints(*block_tables, {rows, width}, "copy_pages", "block_tables"));
  }
  check(mlxq_cache_copy_pages(cache.data(), planes, pages * page, pages, page, page, ints(src, {n}, "copy_pages", "src"),
                              ints(dst, {n}, "copy_pages", "dst"), n, t, rows, width, width, s));
}

}  // namespace mlxq
