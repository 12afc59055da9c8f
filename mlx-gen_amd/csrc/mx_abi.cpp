// mx_abi.cpp — the extern "C" boundary of a decoder block's operators in microscaled types (quantisation, products, norms,
// routing): argument checks and launches.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "mx.h"

using namespace mlxq;

namespace {

int bytes_of(int dtype) { return dtype == MLXQ_FLOAT32 ? 4 : 2; }

int check_dtype(const char* op, const char* what, int dt) {
  if (dt != MLXQ_FLOAT32 && dt != MLXQ_BFLOAT16 && dt != MLXQ_FLOAT16)
    return set_error(MLXQ_EINVAL, "%s: %s %d is not float32, bfloat16 or float16", op, what, dt);
  return MLXQ_OK;
}

int check_ptr(const char* op, const char* what, const void* p, uintptr_t align) {
  if (!p) return set_error(MLXQ_EINVAL, "%s: %s is null", op, what);
  if (reinterpret_cast<uintptr_t>(p) % align != 0)
    return set_error(MLXQ_EINVAL, "%s: %s must be %d-byte aligned", op, what, (int)align);
  return MLXQ_OK;
}

int check_size(const char* op, const char* what, int64_t n, int64_t most) {
  if (n < 0 || n > most) return set_error(MLXQ_EINVAL, "%s: %s=%lld is not from 0 to %lld", op, what, (long long)n, (long long)most);
  return MLXQ_OK;
}

int check_workspace(const char* op, const void* ws, size_t have, size_t need) {
  if (need == 0) return MLXQ_OK;
  if (have < need) return set_error(MLXQ_EINVAL, "%s: a workspace of %zu bytes, %zu are needed", op, have, need);
  return check_ptr(op, "workspace", ws, 16);
}

constexpr int64_t kMostRows = 0x7fffffff - (1 << 20);

int check_k(const char* op, int64_t K) {
  if (K < 32 || K % 32 != 0 || K > 0x7fffff80 - 128)
    return set_error(MLXQ_EINVAL, "%s: K=%lld is not a positive multiple of 32", op, (long long)K);
  return MLXQ_OK;
}

// A microscaled matrix of rows of K; `rows` 0: nothing is read.
int check_mx(const char* op, const char* what, const mlxq_mx* x, int64_t rows, int64_t K) {
  if (!x) return set_error(MLXQ_EINVAL, "%s: %s is null", op, what);
  if (x->format != MLXQ_MX_E2M1 && x->format != MLXQ_MX_E4M3)
    return set_error(MLXQ_EINVAL, "%s: format %d of %s is neither e2m1 nor e4m3", op, x->format, what);
  if (rows == 0) return MLXQ_OK;
  if (int rc = check_ptr(op, what, x->codes, 16)) return rc;
  if (!x->scales || reinterpret_cast<uintptr_t>(x->scales) % 4 != 0)
    return set_error(MLXQ_EINVAL, "%s: the scales of %s must be 4-byte aligned and not null", op, what);
  if (x->scale_stride < K / 32 || x->scale_stride % 4 != 0)
    return set_error(MLXQ_EINVAL, "%s: scale_stride %lld of %s is not a multiple of 4 of at least %lld", op,
                     (long long)x->scale_stride, what, (long long)(K / 32));
  return MLXQ_OK;
}

MxView view(const mlxq_mx* x) { return {(unsigned char*)x->codes, (unsigned char*)x->scales, x->scale_stride}; }

// A [token][head][feature] operand of any element strides; in results (out) no two rows may share memory.
int check_rows(const char* op, const char* what, const mlxq_heads* x, int dtype, int64_t T, int64_t heads, int64_t D, bool out) {
  if (!x) return set_error(MLXQ_EINVAL, "%s: %s is null", op, what);
  if (x->heads != heads) return set_error(MLXQ_EINVAL, "%s: %s has %lld heads, not %lld", op, what, (long long)x->heads, (long long)heads);
  if (int rc = check_ptr(op, what, x->data, bytes_of(dtype))) return rc;
  if (!out) return MLXQ_OK;
  const int64_t none = INT64_MAX / 2, ts = T > 1 ? x->token_stride : none, hs = heads > 1 ? x->head_stride : none;
  const bool apart = ts <= hs ? ts >= D && (ts == none || hs / T >= ts) : hs >= D && ts / heads >= hs;
  if (!apart) return set_error(MLXQ_EINVAL, "%s: tokens or heads of %s overlap", op, what);
  return MLXQ_OK;
}

RowsView view(const mlxq_heads* x) { return x ? RowsView{(unsigned char*)x->data, x->token_stride, x->head_stride} : RowsView{nullptr, 0, 0}; }
// The kernels index by T; 16-bit elements are two bytes there.
int check_norm(const char* op, const mlxq_heads* x, int dtype, int64_t T, int64_t D, const void* weight, int weight_dtype, float eps) {
  int rc;
  if ((rc = check_dtype(op, "dtype", dtype))) return rc;
  if (!x) return set_error(MLXQ_EINVAL, "%s: x is null", op);
  if (x->heads < 1 || x->heads > 0x3fffffff) return set_error(MLXQ_EINVAL, "%s: x has %lld heads", op, (long long)x->heads);
  if (D < 1) return set_error(MLXQ_EINVAL, "%s: D=%lld", op, (long long)D);
  if (D > 32768) return set_error(MLXQ_EUNSUPPORTED, "%s: D=%lld is past 32768", op, (long long)D);
  if (T < 0 || T > kMostRows / x->heads) return set_error(MLXQ_EINVAL, "%s: %lld tokens of %lld heads", op, (long long)T, (long long)x->heads);
  if (!(eps >= 0.0f) || !isfinite(eps)) return set_error(MLXQ_EINVAL, "%s: eps=%g", op, (double)eps);
  if (!weight) return MLXQ_OK;
  if ((rc = check_dtype(op, "weight_dtype", weight_dtype))) return rc;
  return check_ptr(op, "weight", weight, bytes_of(weight_dtype));
}

// Same rows in the same places: an operation may then be in place.
bool same(const mlxq_heads* a, const mlxq_heads* b) {
  return a->data != b->data || (a->token_stride == b->token_stride && a->head_stride == b->head_stride);
}

int check_routing(const char* op, const mlxq_routing* r) {
  if (!r) return set_error(MLXQ_EINVAL, "%s: the routing is null", op);
  if (r->experts < 1 || r->experts > 1024)
    return set_error(r->experts > 1024 ? MLXQ_EUNSUPPORTED : MLXQ_EINVAL, "%s: %lld experts are not from 1 to 1024", op, (long long)r->experts);
  if (r->top_k < 1 || r->top_k > 64)
    return set_error(r->top_k > 64 ? MLXQ_EUNSUPPORTED : MLXQ_EINVAL, "%s: top_k=%lld is not from 1 to 64", op, (long long)r->top_k);
  if (r->tokens < 0 || r->tokens > kMostRows / r->top_k)
    return set_error(MLXQ_EINVAL, "%s: %lld tokens of %lld choices", op, (long long)r->tokens, (long long)r->top_k);
  if (r->tokens == 0) return MLXQ_OK;
  return check_ptr(op, "ids", r->ids, 4);
}

int check_plan(const char* op, const mlxq_routing* r) {
  int rc;
  if ((rc = check_ptr(op, "starts", r->starts, 4))) return rc;
  return r->tokens ? check_ptr(op, "rows", r->rows, 4) : MLXQ_OK;
}

int check_logits(const char* op, const void* logits, int dtype, int64_t row_stride, const mlxq_router* r, const mlxq_routing* o) {
  int rc;
  if ((rc = check_dtype(op, "dtype", dtype))) return rc;
  if (!r) return set_error(MLXQ_EINVAL, "%s: the router is null", op);
  if (r->scoring != MLXQ_ROUTE_SOFTMAX && r->scoring != MLXQ_ROUTE_SIGMOID)
    return set_error(MLXQ_EINVAL, "%s: scoring %d is neither softmax nor sigmoid", op, r->scoring);
  if (!isfinite(r->scale)) return set_error(MLXQ_EINVAL, "%s: scale=%g", op, (double)r->scale);
  if (o->tokens == 0) return MLXQ_OK;
  (void)row_stride;  // any: rows of logits may be a broadcast or a reversal
  return check_ptr(op, "logits", logits, bytes_of(dtype));
}

}  // namespace

extern "C" {

int mlxq_mx_quantize(const void* x, int dtype, int64_t rows, int64_t K, int64_t row_stride, const mlxq_mx* out, void* stream) {
  const char* op = "mx_quantize";
  int rc;
  if ((rc = check_dtype(op, "dtype", dtype)) || (rc = check_size(op, "rows", rows, kMostRows)) || (rc = check_k(op, K)) ||
      (rc = check_mx(op, "out", out, rows, K)))
    return rc;
  if (rows == 0) return MLXQ_OK;
  if ((rc = check_ptr(op, "x", x, 16))) return rc;
  if (rows > 1 && row_stride * bytes_of(dtype) % 16 != 0)
    return set_error(MLXQ_EINVAL, "%s: rows of x must start at multiples of 16 bytes", op);
  return run_mx_quantize(x, dtype, rows, K, row_stride, view(out), out->format, (hipStream_t)stream);
}

int mlxq_mx_dequantize(const mlxq_mx* x, int64_t rows, int64_t K, void* out, int out_dtype, void* stream) {
  const char* op = "mx_dequantize";
  int rc;
  if ((rc = check_dtype(op, "out_dtype", out_dtype)) || (rc = check_size(op, "rows", rows, kMostRows)) || (rc = check_k(op, K)) ||
      (rc = check_mx(op, "x", x, rows, K)))
    return rc;
  if (rows == 0) return MLXQ_OK;
  if ((rc = check_ptr(op, "out", out, 16))) return rc;
  return run_mx_dequantize(view(x), x->format, rows, K, out, out_dtype, (hipStream_t)stream);
}

int mlxq_mx_matmul(const mlxq_mx* x, int64_t M, int64_t K, const mlxq_mx* w, int64_t N, const void* bias, int bias_dtype, void* y,
                   int y_dtype, void* stream) {
  const char* op = "mx_matmul";
  int rc;
  if ((rc = check_size(op, "M", M, kMostRows)) || (rc = check_size(op, "N", N, kMostRows)) || (rc = check_k(op, K)) ||
      (rc = check_mx(op, "x", x, M, K)) || (rc = check_mx(op, "w", w, N, K)) || (rc = check_dtype(op, "y_dtype", y_dtype)))
    return rc;
  if (w->format != MLXQ_MX_E2M1) return set_error(MLXQ_EUNSUPPORTED, "%s: weights must be e2m1", op);
  if (bias && ((rc = check_dtype(op, "bias_dtype", bias_dtype)) || (rc = check_ptr(op, "bias", bias, bytes_of(bias_dtype))))) return rc;
  if (M == 0 || N == 0) return MLXQ_OK;
  if ((rc = check_ptr(op, "y", y, bytes_of(y_dtype)))) return rc;
  MxProduct p = {};
  p.x = view(x);
  p.w = view(w);
  p.M = M;
  p.N = N;
  p.K = K;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.y = y;
  p.y_dtype = y_dtype;
  return run_mx_product(p, x->format, (hipStream_t)stream);
}

int mlxq_rms_norm(const mlxq_heads* x, int dtype, int64_t T, int64_t D, const mlxq_heads* residual, const mlxq_heads* sum,
                  const void* weight, int weight_dtype, float eps, const mlxq_heads* y, const mlxq_mx* y_mx, void* stream) {
  const char* op = "rms_norm";
  int rc;
  if ((rc = check_norm(op, x, dtype, T, D, weight, weight_dtype, eps))) return rc;
  if (!y == !y_mx) return set_error(MLXQ_EINVAL, "%s: one of y and y_mx is needed", op);
  if (!residual != !sum) return set_error(MLXQ_EINVAL, "%s: residual and sum come together", op);
  const int64_t H = x->heads;
  if (y_mx) {
    if (D % 32 != 0) return set_error(MLXQ_EINVAL, "%s: D=%lld is not a multiple of 32", op, (long long)D);
    if ((rc = check_mx(op, "y_mx", y_mx, T, D))) return rc;
    if (y_mx->format != MLXQ_MX_E4M3) return set_error(MLXQ_EUNSUPPORTED, "%s: an 8-bit result is e4m3", op);
  }
  if (T == 0) return MLXQ_OK;
  if ((rc = check_rows(op, "x", x, dtype, T, H, D, false)) || (residual && (rc = check_rows(op, "residual", residual, dtype, T, H, D, false))) ||
      (sum && (rc = check_rows(op, "sum", sum, dtype, T, H, D, true))) || (y && (rc = check_rows(op, "y", y, dtype, T, H, D, true))))
    return rc;
  if ((sum && (!same(sum, x) || !same(sum, residual))) || (y && !same(y, x)) || (y && sum && y->data == sum->data))
    return set_error(MLXQ_EINVAL, "%s: results in place must have their operand's strides, and y is not the sum", op);
  NormArgs a = {};
  a.x = view(x);
  a.res = view(residual);
  a.sum = view(sum);
  a.y = view(y);
  if (y_mx) a.mx = view(y_mx);
  a.w = weight;
  a.w_dtype = weight ? weight_dtype : -1;
  a.eps = eps;
  a.rows = T * H;
  a.heads = (int)H;
  a.D = (int)D;
  a.by_heads = Divisor(H);
  return run_rms_norm(a, dtype, (hipStream_t)stream);
}

size_t mlxq_rms_norm_backward_workspace_size(int64_t T, int64_t heads, int64_t D, int dtype) {
  if (T < 1 || heads < 1 || D < 1 || D > 32768 || T > kMostRows / heads) return 0;
  return (size_t)norm_grad_parts(T * heads, D, dtype) * D * 4;
}

int mlxq_rms_norm_backward(const mlxq_heads* dy, const mlxq_heads* x, int dtype, int64_t T, int64_t D, const void* weight,
                           int weight_dtype, const mlxq_heads* dsum, float eps, const mlxq_heads* dx, void* dweight,
                           void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "rms_norm_backward";
  int rc;
  if ((rc = check_norm(op, x, dtype, T, D, weight, weight_dtype, eps))) return rc;
  if (!weight != !dweight) return set_error(MLXQ_EINVAL, "%s: weight and dweight come together", op);
  if (dweight && (rc = check_ptr(op, "dweight", dweight, bytes_of(weight_dtype)))) return rc;
  const int64_t H = x->heads;
  if (T > 0 && ((rc = check_rows(op, "x", x, dtype, T, H, D, false)) || (rc = check_rows(op, "dy", dy, dtype, T, H, D, false)) ||
                (dsum && (rc = check_rows(op, "dsum", dsum, dtype, T, H, D, false))) || (rc = check_rows(op, "dx", dx, dtype, T, H, D, true))))
    return rc;
  if (T > 0 && (!same(dx, dy) || (dsum && !same(dx, dsum)) || dx->data == x->data))
    return set_error(MLXQ_EINVAL, "%s: dx in place must have its operand's strides, and is not x", op);
  NormGradArgs a = {};
  a.w = weight;
  a.w_dtype = weight ? weight_dtype : -1;
  a.dw = dweight;
  a.eps = eps;
  a.rows = T * H;
  a.heads = (int)H;
  a.D = (int)D;
  a.by_heads = Divisor(H);
  if (T == 0) return run_rms_norm_backward(a, dtype, (hipStream_t)stream);  // no rows: dweight is 0
  const size_t need = mlxq_rms_norm_backward_workspace_size(T, H, D, dtype);
  if (weight && (rc = check_workspace(op, workspace, workspace_bytes, need))) return rc;
  a.dy = view(dy);
  a.x = view(x);
  a.dsum = view(dsum);
  a.dx = view(dx);
  a.part = (float*)workspace;
  a.parts = (int)norm_grad_parts(a.rows, D, dtype);
  return run_rms_norm_backward(a, dtype, (hipStream_t)stream);
}

size_t mlxq_route_workspace_size(int64_t choices, int64_t experts) {
  if (choices < 1 || experts < 1 || experts > 1024 || choices > kMostRows) return 0;
  return route_plan_workspace(choices, experts);
}

static RouteArgs route_args(const void* logits, int64_t row_stride, const mlxq_router* r, const mlxq_routing* o) {
  RouteArgs a = {};
  a.logits = logits;
  a.row_stride = row_stride;
  a.T = (int)o->tokens;
  a.E = (int)o->experts;
  a.k = (int)o->top_k;
  a.scoring = r->scoring;
  a.groups = a.kept = a.best = 1;
  a.normalize = r->normalize;
  a.scale = r->scale;
  a.ids = o->ids;
  a.weights = o->weights;
  return a;
}

int mlxq_route_experts(const void* logits, int dtype, int64_t row_stride, const mlxq_router* router, const uint8_t* active,
                       const mlxq_routing* out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "route_experts";
  int rc;
  if ((rc = check_routing(op, out)) || (rc = check_logits(op, logits, dtype, row_stride, router, out)) || (rc = check_plan(op, out))) return rc;
  const int64_t E = out->experts, G = router->groups;
  if (router->top_k != out->top_k) return set_error(MLXQ_EINVAL, "%s: top_k of router and routing differ", op);
  if (G < 1 || G > 64 || E % G != 0) return set_error(MLXQ_EINVAL, "%s: %lld experts in %lld groups", op, (long long)E, (long long)G);
  if (router->kept_groups < 1 || router->kept_groups > G)
    return set_error(MLXQ_EINVAL, "%s: kept_groups=%lld of %lld", op, (long long)router->kept_groups, (long long)G);
  if (router->group_best != 1 && router->group_best != 2)
    return set_error(MLXQ_EINVAL, "%s: group_best=%lld is neither 1 nor 2", op, (long long)router->group_best);
  if (out->top_k > router->kept_groups * (E / G))
    return set_error(MLXQ_EINVAL, "%s: top_k=%lld of %lld experts in the kept groups", op, (long long)out->top_k,
                     (long long)(router->kept_groups * (E / G)));
  if (router->bias && (rc = check_ptr(op, "bias", router->bias, 4))) return rc;
  if (out->tokens > 0 && (rc = check_ptr(op, "weights", out->weights, 4))) return rc;
  const int64_t n = out->tokens * out->top_k;
  if ((rc = check_workspace(op, workspace, workspace_bytes, mlxq_route_workspace_size(n, E)))) return rc;
  if (out->tokens > 0) {
    RouteArgs a = route_args(logits, row_stride, router, out);
    a.groups = (int)G;
    a.kept = (int)router->kept_groups;
    a.best = (int)router->group_best;
    a.bias = router->bias;
    a.active = active;
    if ((rc = run_route(a, dtype, (hipStream_t)stream))) return rc;
  }
  return run_route_plan(out->ids, n, E, out->starts, out->rows, workspace, (hipStream_t)stream);
}

int mlxq_route_plan(const mlxq_routing* out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "route_plan";
  int rc;
  if ((rc = check_routing(op, out)) || (rc = check_plan(op, out))) return rc;
  const int64_t n = out->tokens * out->top_k;
  if ((rc = check_workspace(op, workspace, workspace_bytes, mlxq_route_workspace_size(n, out->experts)))) return rc;
  return run_route_plan(out->ids, n, out->experts, out->starts, out->rows, workspace, (hipStream_t)stream);
}

int mlxq_route_experts_backward(const float* dweights, const void* logits, int dtype, int64_t row_stride, const mlxq_router* router,
                                const mlxq_routing* routing, void* dlogits, void* stream) {
  const char* op = "route_experts_backward";
  int rc;
  if ((rc = check_routing(op, routing)) || (rc = check_logits(op, logits, dtype, row_stride, router, routing))) return rc;
  if (routing->tokens == 0) return MLXQ_OK;
  if ((rc = check_ptr(op, "dweights", dweights, 4)) || (rc = check_ptr(op, "dlogits", dlogits, bytes_of(dtype)))) return rc;
  return run_route_backward(route_args(logits, row_stride, router, routing), dtype, dweights, dlogits, (hipStream_t)stream);
}

// Workspace of mlxq_mx_experts: the products before they are summed.
size_t mlxq_mx_experts_workspace_size(int64_t tokens, int64_t top_k, int64_t N, int combine, int y_dtype) {
  if (!combine || tokens < 1 || top_k < 1 || N < 1 || tokens > kMostRows / top_k || N > kMostRows) return 0;
  return (size_t)(tokens * top_k) * (size_t)N * bytes_of(y_dtype);
}

int mlxq_mx_experts(const mlxq_mx* x, int x_per_choice, int64_t K, const mlxq_mx* w, int64_t N, const void* bias, int bias_dtype,
                    const mlxq_routing* routing, int combine, void* y, int y_dtype, void* workspace, size_t workspace_bytes,
                    void* stream) {
  const char* op = "mx_experts";
  int rc;
  if ((rc = check_routing(op, routing)) || (rc = check_plan(op, routing)) || (rc = check_size(op, "N", N, kMostRows / routing->experts)) ||
      (rc = check_k(op, K)))
    return rc;
  const int64_t T = routing->tokens, k = routing->top_k, E = routing->experts;
  if ((rc = check_mx(op, "x", x, T, K)) || (rc = check_mx(op, "w", w, E * N, K)) || (rc = check_dtype(op, "y_dtype", y_dtype))) return rc;
  if (w->format != MLXQ_MX_E2M1) return set_error(MLXQ_EUNSUPPORTED, "%s: weights must be e2m1", op);
  if (bias && ((rc = check_dtype(op, "bias_dtype", bias_dtype)) || (rc = check_ptr(op, "bias", bias, bytes_of(bias_dtype))))) return rc;
  if (T == 0 || N == 0) return MLXQ_OK;
  if ((rc = check_ptr(op, "y", y, bytes_of(y_dtype)))) return rc;
  if (combine && (rc = check_ptr(op, "weights", routing->weights, 4))) return rc;
  const size_t need = mlxq_mx_experts_workspace_size(T, k, N, combine, y_dtype);
  if ((rc = check_workspace(op, workspace, workspace_bytes, need))) return rc;
  MxProduct p = {};
  p.x = view(x);
  p.w = view(w);
  p.M = T * k;
  p.N = N;
  p.K = K;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.y = combine ? workspace : y;
  p.y_dtype = y_dtype;
  p.E = (int)E;
  p.starts = routing->starts;
  p.rows = routing->rows;
  p.skip_none = combine != 0;  // the sum leaves them out
  p.by_choices = Divisor(x_per_choice ? 1 : k);
  if ((rc = run_mx_product(p, x->format, (hipStream_t)stream))) return rc;
  if (!combine) return MLXQ_OK;
  return run_mx_combine(workspace, y_dtype, routing->ids, routing->weights, T, k, E, N, y, (hipStream_t)stream);
}

}  // extern "C"
