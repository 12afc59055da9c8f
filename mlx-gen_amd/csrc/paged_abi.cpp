// paged_abi.cpp — the extern "C" boundary of the paged-cache operators: argument checks and launches.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "paged.h"

using namespace mlxq;

namespace {

int bytes_of(int dtype) { return dtype == MLXQ_FLOAT32 ? 4 : 2; }

int check_dtype(const char* op, int dt) {
  if (dt != MLXQ_FLOAT32 && dt != MLXQ_BFLOAT16 && dt != MLXQ_FLOAT16)
    return set_error(MLXQ_EINVAL, "%s: dtype %d is not float32, bfloat16 or float16", op, dt);
  return MLXQ_OK;
}

int check_ptr(const char* op, const char* what, const void* p, uintptr_t align) {
  if (!p) return set_error(MLXQ_EINVAL, "%s: %s is null", op, what);
  if (reinterpret_cast<uintptr_t>(p) % align != 0)
    return set_error(MLXQ_EINVAL, "%s: %s must be %d-byte aligned", op, what, (int)align);
  return MLXQ_OK;
}

// A [token][head][feature] operand whose heads are read in 16-byte pieces.  Strides may be 0 or negative in
// inputs (a broadcast, a reversal); in results (tokens > 0 gives their number) no two heads may share memory.
int check_heads(const char* op, const char* what, const mlxq_heads* x, int dtype, int64_t D, int64_t tokens = 0) {
  if (!x) return set_error(MLXQ_EINVAL, "%s: %s is null", op, what);
  int rc;
  if ((rc = check_ptr(op, what, x->data, 16))) return rc;
  const int64_t C = 16 / bytes_of(dtype);
  if (x->heads < 1 || x->heads > 65535) return set_error(MLXQ_EINVAL, "%s: %s has %lld heads", op, what, (long long)x->heads);
  if (x->token_stride % C != 0 || x->head_stride % C != 0)
    return set_error(MLXQ_EINVAL, "%s: strides of %s must be multiples of 16 bytes", op, what);
  if (tokens == 0) return MLXQ_OK;
  const int64_t ts = tokens > 1 ? x->token_stride : INT64_MAX / 2, hs = x->heads > 1 ? x->head_stride : INT64_MAX / 2;
  const bool apart = ts <= hs ? ts >= D && (ts == INT64_MAX / 2 || hs / tokens >= ts) : hs >= D && ts / x->heads >= hs;
  if (!apart) return set_error(MLXQ_EINVAL, "%s: tokens or heads of %s overlap", op, what);
  return MLXQ_OK;
}

int check_rotary(const char* op, const float* table, int64_t rows, int64_t R, int64_t D) {
  if (R < 0 || R > 256 || R % 2 != 0 || R > D)
    return set_error(MLXQ_EINVAL, "%s: rotary_dim %lld must be even, at most 256 and at most head_dim=%lld", op, (long long)R,
                     (long long)D);
  if (R == 0) return MLXQ_OK;
  if (rows < 1 || rows > 0x7fffffff) return set_error(MLXQ_EINVAL, "%s: a table of %lld positions", op, (long long)rows);
  return check_ptr(op, "table", table, 16);
}

int check_cache(const char* op, const mlxq_paged_cache* c, int64_t T) {
  if (!c) return set_error(MLXQ_EINVAL, "%s: cache is null", op);
  int rc;
  if ((rc = check_dtype(op, c->dtype))) return rc;
  if (c->heads < 1 || c->heads > 65535) return set_error(MLXQ_EINVAL, "%s: the cache has %lld heads", op, (long long)c->heads);
  if (c->head_dim < 16 || c->head_dim % 16 != 0 || c->head_dim > 256)
    return set_error(MLXQ_EUNSUPPORTED, "%s: head_dim %lld is not a multiple of 16 up to 256", op, (long long)c->head_dim);
  const int64_t P = c->page_size;
  if (P < 16 || P > 1024 || (P & (P - 1)) != 0)
    return set_error(MLXQ_EINVAL, "%s: page_size %lld is not a power of two from 16 to 1024", op, (long long)P);
  if (c->pages < 0 || c->pages > 0x7fffffff) return set_error(MLXQ_EINVAL, "%s: a pool of %lld pages", op, (long long)c->pages);
  if (T == 0) return MLXQ_OK;
  if (c->pages == 0) return set_error(MLXQ_EINVAL, "%s: the cache has no pages", op);
  if ((rc = check_ptr(op, "k cache", c->k, 16)) || (rc = check_ptr(op, "v cache", c->v, 16))) return rc;
  const int64_t n = c->heads * P * c->head_dim, C = 16 / bytes_of(c->dtype);
  if (c->k_page_stride < n || c->v_page_stride < n || c->k_page_stride % C != 0 || c->v_page_stride % C != 0)
    return set_error(MLXQ_EINVAL, "%s: page strides must be multiples of 16 bytes and at least a page's %lld elements", op,
                     (long long)n);
  return MLXQ_OK;
}

int check_batch(const char* op, const mlxq_paged_batch* b, int64_t T) {
  if (!b) return set_error(MLXQ_EINVAL, "%s: batch is null", op);
  if (T < 0 || T > 0x3fffffff) return set_error(MLXQ_EINVAL, "%s: T=%lld", op, (long long)T);
  if (b->sequences < 0 || b->sequences > 0xffffff || b->table_width < 0 || b->table_width > 0x7fffffff)
    return set_error(MLXQ_EINVAL, "%s: block tables of [%lld, %lld]", op, (long long)b->sequences, (long long)b->table_width);
  if (b->max_q < 0 || b->max_kv < 0) return set_error(MLXQ_EINVAL, "%s: max_q and max_kv must not be negative", op);
  if (T == 0 || b->sequences == 0) return MLXQ_OK;
  int rc;
  if (b->sequences > 1 && b->table_stride < b->table_width)
    return set_error(MLXQ_EINVAL, "%s: rows of the block tables overlap", op);
  if (b->table_width > 0 && (rc = check_ptr(op, "block_tables", b->block_tables, 4))) return rc;
  if ((rc = check_ptr(op, "q_starts", b->q_starts, 4))) return rc;
  return check_ptr(op, "kv_lens", b->kv_lens, 4);
}

// A window as the kernels and their plan count it: past every place it hides nothing.
int64_t window_of(const mlxq_attention* o) { return std::min<int64_t>(o->window, 0x3fffffff); }

Heads view(const mlxq_heads* x) { return {x->data, x->token_stride, x->head_stride}; }

Batch view(const mlxq_paged_batch* b, const mlxq_paged_cache* c, int64_t T) {
  Batch r = {};
  r.tables = b->block_tables;
  r.q_starts = b->q_starts;
  r.kv_lens = b->kv_lens;
  r.table_stride = b->table_stride;
  r.B = (int)b->sequences;
  r.T = (int)T;
  while ((1 << r.page_log2) < c->page_size) ++r.page_log2;
  // Places with a page are kept below 2^30, so that a place plus a tile never passes 31 bits.
  r.capacity = (int)std::min<int64_t>(b->table_width * c->page_size, 0x3ffffff0);
  r.pages = (int)c->pages;
  return r;
}

int check_attention(const char* op, int64_t T, int64_t q_heads, const mlxq_paged_cache* cache, const mlxq_paged_batch* batch,
                    const mlxq_attention* o) {
  int rc;
  if ((rc = check_batch(op, batch, T)) || (rc = check_cache(op, cache, T))) return rc;
  if (q_heads < 1 || q_heads > 65535 || q_heads % cache->heads != 0)
    return set_error(MLXQ_EINVAL, "%s: %lld query heads over %lld key heads", op, (long long)q_heads, (long long)cache->heads);
  // A sequence's rows, (token, query head) pairs of a key head, and a tile of 128 past them are counted in 31 bits.
  if (T * (q_heads / cache->heads) > 0x7fffffff - 128)
    return set_error(MLXQ_EINVAL, "%s: %lld tokens of %lld query heads a key head are too many rows", op, (long long)T,
                     (long long)(q_heads / cache->heads));
  if (!o) return set_error(MLXQ_EINVAL, "%s: options are null", op);
  if (!(o->scale > 0.0f) || !isfinite(o->scale)) return set_error(MLXQ_EINVAL, "%s: scale must be positive and finite", op);
  if (!(o->softcap >= 0.0f) || !isfinite(o->softcap))
    return set_error(MLXQ_EINVAL, "%s: softcap must be finite and not negative", op);
  if (o->window < 0) return set_error(MLXQ_EINVAL, "%s: window must not be negative", op);
  const struct {
    const void* p;
    const char* what;
  } arrays[] = {{o->prefix_lens, "prefix_lens"}, {o->alibi_slopes, "alibi_slopes"}, {o->sinks, "sinks"}};
  for (const auto& a : arrays)
    if (a.p && (rc = check_ptr(op, a.what, a.p, 4))) return rc;
  return MLXQ_OK;
}

// The plan of a checked call, unless its workgroups pass what a launch has.
int plan_of(const char* op, int64_t T, int64_t q_heads, const mlxq_paged_cache* c, const mlxq_paged_batch* b,
            const mlxq_attention* o, AttnPlan& plan) {
  const int64_t capacity = b->table_width * c->page_size;
  const int64_t max_q = std::min<int64_t>(std::max<int64_t>(b->max_q, 1), 0x3fffffff);
  plan = plan_attention(T, q_heads, c->heads, c->head_dim, c->dtype, b->sequences, max_q,
                        std::min(std::max<int64_t>(b->max_kv, 1), std::max<int64_t>(capacity, 1)), window_of(o), o->causal != 0);
  if (plan.blocks > most_groups(256)) return set_error(MLXQ_EINVAL, "%s: problem too large", op);
  return MLXQ_OK;
}

}  // namespace

extern "C" {

int mlxq_rotary_frequencies(int64_t rotary_dim, double base, const mlxq_rope_scaling* s, double* inv_freq,
                            double* magnitude) {
  set_error(MLXQ_OK, "%s", "");
  const char* op = "rotary_frequencies";
  if (rotary_dim < 2 || rotary_dim > 256 || rotary_dim % 2 != 0)
    return set_error(MLXQ_EINVAL, "%s: rotary_dim %lld must be even, from 2 to 256", op, (long long)rotary_dim);
  if (!(base > 1.0) || !isfinite(base)) return set_error(MLXQ_EINVAL, "%s: base must be finite and above 1", op);
  if (!inv_freq || !magnitude) return set_error(MLXQ_EINVAL, "%s: a result is null", op);
  const int kind = s ? s->kind : MLXQ_ROPE_NONE;
  if (kind < MLXQ_ROPE_NONE || kind > MLXQ_ROPE_LLAMA3) return set_error(MLXQ_EINVAL, "%s: unknown scaling %d", op, kind);
  const double r = (double)rotary_dim, pi2 = 2.0 * 3.14159265358979323846;
  if (kind != MLXQ_ROPE_NONE && (!(s->factor >= 1.0) || !isfinite(s->factor)))
    return set_error(MLXQ_EINVAL, "%s: factor must be finite and at least 1", op);
  if (kind == MLXQ_ROPE_NTK && rotary_dim == 2)
    return set_error(MLXQ_EINVAL, "%s: the ntk scaling needs more than one pair", op);
  if (kind == MLXQ_ROPE_YARN || kind == MLXQ_ROPE_LLAMA3) {
    if (!(s->original_context > 0.0) || !isfinite(s->original_context))
      return set_error(MLXQ_EINVAL, "%s: original_context must be positive", op);
    if (!(s->low > 0.0) || !(s->high > s->low) || !isfinite(s->high))
      return set_error(MLXQ_EINVAL, "%s: bounds must satisfy 0 < low < high", op);
  }
  if (kind == MLXQ_ROPE_NTK) base *= pow(s->factor, r / (r - 2.0));
  *magnitude = kind == MLXQ_ROPE_YARN ? 0.1 * log(s->factor) + 1.0 : 1.0;
  const int64_t half = rotary_dim / 2;
  double from = 0.0, to = 1.0;
  if (kind == MLXQ_ROPE_YARN) {
    // The pair index at which a wave turns n times over the trained context.
    auto index = [&](double n) { return r * log(s->original_context / (n * pi2)) / (2.0 * log(base)); };
    from = std::max(floor(index(s->high)), 0.0);
    to = std::min(ceil(index(s->low)), r - 1.0);
    if (!(to > from)) to = from + 0.001;
  }
  for (int64_t i = 0; i < half; ++i) {
    double f = pow(base, -2.0 * (double)i / r);
    if (kind == MLXQ_ROPE_LINEAR) f /= s->factor;
    if (kind == MLXQ_ROPE_YARN) {
      const double ramp = std::min(std::max(((double)i - from) / (to - from), 0.0), 1.0);
      f = f / s->factor * ramp + f * (1.0 - ramp);
    }
    if (kind == MLXQ_ROPE_LLAMA3) {
      const double n = s->original_context * f / pi2;
      const double keep = std::min(std::max((n - s->low) / (s->high - s->low), 0.0), 1.0);
      f = f / s->factor * (1.0 - keep) + f * keep;
    }
    inv_freq[i] = f;
  }
  return MLXQ_OK;
}

int mlxq_rotary_table(const double* inv_freq, int64_t rotary_dim, double magnitude, int64_t positions, float* table,
                      void* stream) {
  set_error(MLXQ_OK, "%s", "");
  const char* op = "rotary_table";
  if (rotary_dim < 2 || rotary_dim > 256 || rotary_dim % 2 != 0)
    return set_error(MLXQ_EINVAL, "%s: rotary_dim %lld must be even, from 2 to 256", op, (long long)rotary_dim);
  if (!inv_freq) return set_error(MLXQ_EINVAL, "%s: inv_freq is null", op);
  if (positions < 0) return set_error(MLXQ_EINVAL, "%s: positions=%lld < 0", op, (long long)positions);
  if (positions == 0) return MLXQ_OK;
  if (int rc = check_ptr(op, "table", table, 16)) return rc;
  return run_rotary_table(inv_freq, rotary_dim / 2, magnitude, positions, table, (hipStream_t)stream);
}

int mlxq_rotary(const mlxq_heads* x, int dtype, int64_t T, int64_t head_dim, const int32_t* positions, const float* table,
                int64_t table_rows, int64_t rotary_dim, int interleaved, int inverse, const mlxq_heads* y, void* stream) {
  set_error(MLXQ_OK, "%s", "");
  const char* op = "rotary";
  int rc;
  if ((rc = check_dtype(op, dtype))) return rc;
  if (T < 0 || T > 0x3fffffff) return set_error(MLXQ_EINVAL, "%s: T=%lld", op, (long long)T);
  if (head_dim < 1 || head_dim > 65536 || head_dim * bytes_of(dtype) % 16 != 0)
    return set_error(MLXQ_EINVAL, "%s: head_dim %lld is not a multiple of 16 bytes", op, (long long)head_dim);
  if (rotary_dim == 0) return set_error(MLXQ_EINVAL, "%s: rotary_dim is 0", op);
  if ((rc = check_rotary(op, table, table_rows, rotary_dim, head_dim))) return rc;
  if (T == 0) return MLXQ_OK;
  if ((rc = check_heads(op, "x", x, dtype, head_dim)) || (rc = check_heads(op, "y", y, dtype, head_dim, T)) ||
      (rc = check_ptr(op, "positions", positions, 4)))
    return rc;
  if (x->heads != y->heads) return set_error(MLXQ_EINVAL, "%s: x and y have different heads", op);
  if (x->data == y->data && (x->token_stride != y->token_stride || x->head_stride != y->head_stride))
    return set_error(MLXQ_EINVAL, "%s: in place, x and y must have the same strides", op);
  const RotaryArgs r = {table, positions, (int)table_rows, (int)rotary_dim, interleaved != 0, inverse != 0};
  return run_rotary(view(x), dtype, T, x->heads, head_dim, r, view(y), (hipStream_t)stream);
}

int mlxq_cache_append(const mlxq_heads* k, const mlxq_heads* v, int64_t T, const mlxq_paged_cache* cache,
                      const mlxq_paged_batch* batch, const int32_t* positions, const float* table, int64_t table_rows,
                      int64_t rotary_dim, int interleaved, const mlxq_heads* q, const mlxq_heads* q_out, void* stream) {
  set_error(MLXQ_OK, "%s", "");
  const char* op = "cache_append";
  int rc;
  if ((rc = check_batch(op, batch, T)) || (rc = check_cache(op, cache, T))) return rc;
  const int64_t D = cache->head_dim;
  if ((rc = check_rotary(op, table, table_rows, rotary_dim, D))) return rc;
  if (positions && (rc = check_ptr(op, "positions", positions, 4))) return rc;
  if ((q == nullptr) != (q_out == nullptr)) return set_error(MLXQ_EINVAL, "%s: q and q_out come together", op);
  if (T == 0 || batch->sequences == 0) return MLXQ_OK;
  if ((rc = check_heads(op, "k", k, cache->dtype, D)) || (rc = check_heads(op, "v", v, cache->dtype, D))) return rc;
  if (k->heads != cache->heads || v->heads != cache->heads)
    return set_error(MLXQ_EINVAL, "%s: k and v must have the cache's %lld heads", op, (long long)cache->heads);
  if (q) {
    if ((rc = check_heads(op, "q", q, cache->dtype, D)) ||
        (rc = check_heads(op, "q_out", q_out, cache->dtype, D, T)))
      return rc;
    if (q->heads != q_out->heads || q->heads % cache->heads != 0)
      return set_error(MLXQ_EINVAL, "%s: %lld query heads (%lld in q_out) over %lld key heads", op, (long long)q->heads,
                       (long long)q_out->heads, (long long)cache->heads);
    if (q->data == q_out->data && (q->token_stride != q_out->token_stride || q->head_stride != q_out->head_stride))
      return set_error(MLXQ_EINVAL, "%s: in place, q and q_out must have the same strides", op);
  }
  AppendArgs a = {};
  a.k = view(k);
  a.v = view(v);
  if (q) {
    a.q = view(q);
    a.q_out = view(q_out);
    a.Hq = (int)q->heads;
  }
  a.k_cache = cache->k;
  a.v_cache = cache->v;
  a.k_page = cache->k_page_stride;
  a.v_page = cache->v_page_stride;
  a.batch = view(batch, cache, T);
  a.rot = {rotary_dim ? table : nullptr, positions, (int)table_rows, (int)rotary_dim, interleaved != 0, 0};
  a.Hkv = (int)cache->heads;
  a.D = (int)D;
  // A token each: a sequence is a unit.  Else a sequence of n tokens lies in at most n / 16 + 2 blocks.
  a.direct = batch->max_q <= 1;
  const int64_t units = a.direct ? batch->sequences : T / 16 + 2 * std::min(batch->sequences, T);
  if (units * cache->heads > most_groups(256)) return set_error(MLXQ_EINVAL, "%s: problem too large", op);
  return run_cache_append(a, cache->dtype, units, (hipStream_t)stream);
}

size_t mlxq_paged_attention_workspace_size(int64_t T, int64_t q_heads, const mlxq_paged_cache* cache,
                                           const mlxq_paged_batch* batch, const mlxq_attention* options) {
  const char* op = "paged_attention";
  AttnPlan plan;
  if (check_attention(op, T, q_heads, cache, batch, options) || T == 0 || batch->sequences == 0 ||
      plan_of(op, T, q_heads, cache, batch, options, plan))
    return 0;
  return plan.total;
}

int mlxq_paged_attention(const mlxq_heads* q, int64_t T, const mlxq_paged_cache* cache, const mlxq_paged_batch* batch,
                         const mlxq_attention* o, const mlxq_heads* out, void* workspace, size_t workspace_bytes,
                         void* stream) {
  set_error(MLXQ_OK, "%s", "");
  const char* op = "paged_attention";
  int rc;
  if (!q || !out) return set_error(MLXQ_EINVAL, "%s: q or out is null", op);
  if ((rc = check_attention(op, T, q->heads, cache, batch, o))) return rc;
  if (T == 0 || batch->sequences == 0) return MLXQ_OK;
  const int64_t D = cache->head_dim;
  if ((rc = check_heads(op, "q", q, cache->dtype, D)) || (rc = check_heads(op, "out", out, cache->dtype, D, T)))
    return rc;
  if (out->heads != q->heads) return set_error(MLXQ_EINVAL, "%s: q and out have different heads", op);
  AttnPlan plan;
  if ((rc = plan_of(op, T, q->heads, cache, batch, o, plan))) return rc;
  if (plan.total > 0) {
    if (workspace == nullptr || workspace_bytes < plan.total)
      return set_error(MLXQ_EINVAL, "%s: workspace of %zu bytes is smaller than the %zu required", op, workspace_bytes, plan.total);
    if ((rc = check_ptr(op, "workspace", workspace, 16))) return rc;
  }
  AttnArgs a = {};
  a.q = view(q);
  a.out = view(out);
  a.k = cache->k;
  a.v = cache->v;
  a.k_page = cache->k_page_stride;
  a.v_page = cache->v_page_stride;
  a.batch = view(batch, cache, T);
  a.Hkv = (int)cache->heads;
  a.G = (int)(q->heads / cache->heads);
  a.D = (int)D;
  a.S = plan.S;
  a.chunk = plan.chunk;
  a.by_chunk = Divisor(a.chunk);
  a.items = plan.tiled ? (int)plan.blocks : (int)(plan.blocks / plan.S);
  a.by_hkv = Divisor(a.Hkv);
  a.by_g = Divisor(a.G);
  a.by_items = Divisor(a.items);
  const double log2e = 1.44269504088896341;
  a.scale = a.score_scale = (float)(o->scale * log2e);
  if (o->softcap > 0.0f) {
    // Caps past 1e30 are as far out of every score's reach; cap2 and, for small caps, the scale stay finite.
    const double cap = std::min((double)o->softcap, 1e30);
    a.softcap = (float)cap;
    a.cap2 = (float)(cap * log2e);
    a.scale = (float)std::min(2.0 * o->scale / cap * log2e, 3.4e38);
  }
  a.causal = o->causal != 0;
  a.window = (int)window_of(o);
  a.direct = plan.direct;
  a.prefix = o->prefix_lens;
  a.slopes = o->alibi_slopes;
  a.sinks = o->sinks;
  if (plan.total > 0) {
    a.part = (float*)workspace;
    a.ml = (float*)((char*)workspace + plan.ml);
    a.splits = (int*)((char*)workspace + plan.splits);
  }
  return run_attention(a, cache->dtype, plan, (hipStream_t)stream);
}

int mlxq_cache_copy_pages(void* cache, int64_t planes, int64_t plane_stride, int64_t pages, int64_t page_bytes,
                          int64_t page_stride, const int32_t* src, const int32_t* dst, int64_t count, int32_t* tables,
                          int64_t rows, int64_t width, int64_t table_stride, void* stream) {
  set_error(MLXQ_OK, "%s", "");
  const char* op = "copy_pages";
  int rc;
  if (planes < 0 || pages < 0 || pages > 0x7fffffff || count < 0)
    return set_error(MLXQ_EINVAL, "%s: planes=%lld pages=%lld count=%lld", op, (long long)planes, (long long)pages, (long long)count);
  if (page_bytes < 16 || page_bytes % 16 != 0 || page_stride < page_bytes || page_stride % 16 != 0 || plane_stride % 16 != 0)
    return set_error(MLXQ_EINVAL, "%s: page bytes and strides must be multiples of 16, page strides at least a page", op);
  if (planes > 1 && plane_stride < page_bytes) return set_error(MLXQ_EINVAL, "%s: planes overlap", op);
  if (tables && (rows < 0 || width < 0 || (rows > 1 && table_stride < width)))
    return set_error(MLXQ_EINVAL, "%s: block tables of [%lld, %lld]", op, (long long)rows, (long long)width);
  if (count == 0) return MLXQ_OK;
  if ((rc = check_ptr(op, "src", src, 4)) || (rc = check_ptr(op, "dst", dst, 4))) return rc;
  if (planes > 0 && pages > 0 && (rc = check_ptr(op, "cache", cache, 16))) return rc;
  if (tables && rows * width > 0 && (rc = check_ptr(op, "block_tables", tables, 4))) return rc;
  return run_copy_pages(cache, pages > 0 ? planes : 0, plane_stride, pages, page_bytes, page_stride, src, dst, count, tables,
                        rows, width, table_stride, (hipStream_t)stream);
}

}  // extern "C"
