// mx.cpp — the operators of a decoder block in microscaled types in the C++ host API (see mlxq.hpp): shape checks, workspaces
// and the calls of the C ABI.
#include "../../include/mlxq.h"
#include "mlxq.hpp"

namespace mlxq {

namespace {

void check(int status) {
  if (status != MLXQ_OK) throw Error(status, mlxq_last_error());
}
[[noreturn]] void bad(const std::string& op, const std::string& msg) { throw Error(MLXQ_EINVAL, op + ": " + msg); }

int abi_dtype(Dtype dt, const char* op) {
  if (dt == Dtype::Float32) return MLXQ_FLOAT32;
  if (dt == Dtype::Bfloat16) return MLXQ_BFLOAT16;
  if (dt == Dtype::Float16) return MLXQ_FLOAT16;
  bad(op, std::string("expected float32, bfloat16 or float16, got ") + dtype_name(dt));
}

int64_t pitch(int64_t K) { return (K / 32 + 3) / 4 * 4; }

std::vector<int64_t> with_last(const std::vector<int64_t>& shape, int64_t n) {
  std::vector<int64_t> r = shape;
  r.back() = n;
  return r;
}

mlxq_mx view(const Mx& x, const char* op, const char* what) {
  if (x.codes.ndim() < 1 || x.codes.dtype() != Dtype::Uint8 || x.scales.dtype() != Dtype::Uint8)
    bad(op, std::string("codes and scales of ") + what + " must be uint8");
  const int64_t K = x.K();
  if (K == 0 || K % 32 != 0 || x.scales.shape() != with_last(x.codes.shape(), pitch(K)))
    bad(op, std::string("the scales of ") + what + " must be [..., 4 * ceil(K / 128)] for a K that is a multiple of 32");
  return {x.codes.data(), x.scales.data(), pitch(K), x.format};
}

int64_t rows_of(const Array& x) { return x.dim(-1) == 0 ? 0 : x.size() / x.dim(-1); }

Mx empty_mx(const std::vector<int64_t>& shape, int format) {
  const int64_t K = shape.back();
  return {Array::empty(with_last(shape, format == MLXQ_MX_E2M1 ? K / 2 : K), Dtype::Uint8), Array::empty(with_last(shape, pitch(K)), Dtype::Uint8),
          format};
}

const void* bias_of(const std::optional<Array>& b, std::vector<int64_t> shape, const char* op, int& dt) {
  dt = 0;
  if (!b) return nullptr;
  if (b->shape() != shape) bad(op, "the bias has another shape");
  dt = abi_dtype(b->dtype(), op);
  return b->data();
}

// [..., D] as rows of one head.
mlxq_heads flat(const Array& x) { return {x.data(), 1, x.dim(-1), 0}; }

const void* weight_of(const Array* w, int64_t D, const char* op, int& dt) {
  dt = 0;
  if (!w) return nullptr;
  if (w->shape() != std::vector<int64_t>{D}) bad(op, "the weight must have the last dimension's size");
  dt = abi_dtype(w->dtype(), op);
  return w->data();
}

void same_as(const Array& a, const Array& x, const char* op, const char* what) {
  if (a.shape() != x.shape() || a.dtype() != x.dtype()) bad(op, std::string(what) + " must have x's shape and dtype");
}

mlxq_routing routing_of(const Routing& r, int64_t experts, const char* op) {
  if (r.ids.ndim() != 2 || r.ids.dtype() != Dtype::Int32) bad(op, "ids must be int32 [tokens, top_k]");
  const int64_t T = r.ids.dim(0), k = r.ids.dim(1);
  if (r.weights.shape() != r.ids.shape() || r.weights.dtype() != Dtype::Float32) bad(op, "weights must be float32 of ids' shape");
  if (r.starts.shape() != std::vector<int64_t>{experts + 1} || r.starts.dtype() != Dtype::Int32 ||
      r.rows.shape() != std::vector<int64_t>{T * k} || r.rows.dtype() != Dtype::Int32)
    bad(op, "starts must be int32 [experts + 1] and rows int32 [tokens * top_k]");
  return {(int32_t*)r.ids.data(), (float*)r.weights.data(), (int32_t*)r.starts.data(), (int32_t*)r.rows.data(), T, k, experts};
}

}  // namespace

Mx mx_quantize(const Array& x, int format, hipStream_t s) {
  const char* op = "mx_quantize";
  const int dt = abi_dtype(x.dtype(), op);
  if (x.ndim() < 1 || x.dim(-1) == 0 || x.dim(-1) % 32 != 0) bad(op, "the last dimension must be a positive multiple of 32");
  if (format != MLXQ_MX_E2M1 && format != MLXQ_MX_E4M3) bad(op, "the format is neither e2m1 nor e4m3");
  const int64_t K = x.dim(-1);
  Mx out = empty_mx(x.shape(), format);
  const mlxq_mx v = view(out, op, "out");
  check(mlxq_mx_quantize(x.data(), dt, rows_of(x), K, K, &v, s));
  return out;
}

Array mx_dequantize(const Mx& x, Dtype dt, hipStream_t s) {
  const char* op = "mx_dequantize";
  const int code = abi_dtype(dt, op);
  const mlxq_mx v = view(x, op, "x");
  Array out = Array::empty(with_last(x.codes.shape(), x.K()), dt);
  check(mlxq_mx_dequantize(&v, rows_of(out), x.K(), out.data(), code, s));
  return out;
}

void MxLinear::forward_into(const Mx& x, const Array& y, hipStream_t s) const {
  const char* op = "mx_matmul";
  const mlxq_mx xv = view(x, op, "x"), wv = view(w, op, "w");
  if (w.codes.ndim() != 2 || w.K() != x.K()) bad(op, "w must be [N, K] of x's K");
  const int64_t N = w.codes.dim(0), M = rows_of(x.codes);
  if (y.shape() != with_last(x.codes.shape(), N)) bad(op, "y must be [..., N]");
  int bdt;
  const void* b = bias_of(bias, {N}, op, bdt);
  const int ydt = abi_dtype(y.dtype(), op);
  check(mlxq_mx_matmul(&xv, M, x.K(), &wv, N, b, bdt, y.data(), ydt, s));
}

Array MxLinear::forward(const Mx& x, hipStream_t s) const {
  if (w.codes.ndim() != 2 || x.codes.ndim() < 1) bad("mx_matmul", "x must be [..., K] and w [N, K]");
  Array y = Array::empty(with_last(x.codes.shape(), w.codes.dim(0)), out);
  forward_into(x, y, s);
  return y;
}

Normed rms_norm(const Array& x, const Array* weight, const Array* residual, float eps, bool mx, hipStream_t s) {
  const char* op = "rms_norm";
  const int dt = abi_dtype(x.dtype(), op);
  if (x.ndim() < 1 || x.dim(-1) == 0 || (mx && x.dim(-1) % 32 != 0)) bad(op, "the last dimension must be positive, and a multiple of 32 for mx");
  int wdt;
  const void* w = weight_of(weight, x.dim(-1), op, wdt);
  if (residual) same_as(*residual, x, op, "residual");
  Normed r;
  mlxq_heads xv = flat(x), rv = {}, sv = {}, yv = {};
  mlxq_mx mv = {};
  if (residual) {
    r.sum = Array::empty(x.shape(), x.dtype());
    rv = flat(*residual);
    sv = flat(r.sum);
  }
  if (mx) {
    r.mx = empty_mx(x.shape(), MLXQ_MX_E4M3);
    mv = view(r.mx, op, "y");
  } else {
    r.y = Array::empty(x.shape(), x.dtype());
    yv = flat(r.y);
  }
  check(mlxq_rms_norm(&xv, dt, rows_of(x), x.dim(-1), residual ? &rv : nullptr, residual ? &sv : nullptr, w, wdt, eps, mx ? nullptr : &yv,
                      mx ? &mv : nullptr, s));
  return r;
}

std::pair<Array, Array> RmsNormGradient::backward(const Array& dy, const Array& x, const Array* weight, const Array* dsum,
                                                  hipStream_t s) const {
  const char* op = "rms_norm_backward";
  const int dt = abi_dtype(x.dtype(), op);
  if (x.ndim() < 1 || x.dim(-1) == 0) bad(op, "the last dimension must be positive");
  same_as(dy, x, op, "dy");
  if (dsum) same_as(*dsum, x, op, "dsum");
  int wdt;
  const void* w = weight_of(weight, x.dim(-1), op, wdt);
  Array dx = Array::empty(x.shape(), x.dtype()), dw;
  if (weight) dw = Array::empty(weight->shape(), weight->dtype());
  const mlxq_heads yv = flat(dy), xv = flat(x), dv = flat(dx);
  mlxq_heads sv = {};
  if (dsum) sv = flat(*dsum);
  const size_t need = weight ? mlxq_rms_norm_backward_workspace_size(rows_of(x), 1, x.dim(-1), dt) : 0;
  const Array& ws = workspace_.at_least(need);
  check(mlxq_rms_norm_backward(&yv, &xv, dt, rows_of(x), x.dim(-1), w, wdt, dsum ? &sv : nullptr, eps, &dv, weight ? dw.data() : nullptr,
                               ws.data(), ws.nbytes(), s));
  return {dx, dw};
}

Routing Router::forward(const Array& logits, const Array* active, hipStream_t s) const {
  const char* op = "route_experts";
  const int dt = abi_dtype(logits.dtype(), op);
  if (logits.ndim() != 2) bad(op, "logits must be [tokens, experts]");
  const int64_t T = logits.dim(0), E = logits.dim(1);
  if (bias && (bias->shape() != std::vector<int64_t>{E} || bias->dtype() != Dtype::Float32)) bad(op, "the bias must be float32 [experts]");
  if (active && (active->shape() != std::vector<int64_t>{T} || active->dtype() != Dtype::Bool)) bad(op, "active must be bool [tokens]");
  if (top_k < 1 || top_k > 64) bad(op, "top_k is not from 1 to 64");
  const Routing r = {Array::empty({T, top_k}, Dtype::Int32), Array::empty({T, top_k}, Dtype::Float32), Array::empty({E + 1}, Dtype::Int32),
                     Array::empty({T * top_k}, Dtype::Int32)};
  const mlxq_routing out = routing_of(r, E, op);
  const mlxq_router o = {scoring, top_k, bias ? (const float*)bias->data() : nullptr, groups, kept_groups, group_best, normalize, scale};
  const size_t need = mlxq_route_workspace_size(T * top_k, E);
  const Array& ws = workspace_.at_least(need);
  check(mlxq_route_experts(logits.data(), dt, E, &o, active ? (const uint8_t*)active->data() : nullptr, &out, ws.data(), ws.nbytes(), s));
  return r;
}

Routing Router::plan(const Array& ids, const Array& weights, int64_t experts, hipStream_t s) const {
  const char* op = "route_plan";
  if (ids.ndim() != 2 || experts < 1) bad(op, "ids must be [tokens, top_k]");
  const Routing r = {ids, weights, Array::empty({experts + 1}, Dtype::Int32), Array::empty({ids.size()}, Dtype::Int32)};
  const mlxq_routing out = routing_of(r, experts, op);
  const size_t need = mlxq_route_workspace_size(ids.size(), experts);
  const Array& ws = workspace_.at_least(need);
  check(mlxq_route_plan(&out, ws.data(), ws.nbytes(), s));
  return r;
}

Array Router::backward(const Array& dweights, const Array& logits, const Array& ids, hipStream_t s) const {
  const char* op = "route_experts_backward";
  const int dt = abi_dtype(logits.dtype(), op);
  if (logits.ndim() != 2 || ids.ndim() != 2 || ids.dtype() != Dtype::Int32 || ids.dim(0) != logits.dim(0))
    bad(op, "logits must be [tokens, experts] and ids int32 [tokens, top_k]");
  if (dweights.shape() != ids.shape() || dweights.dtype() != Dtype::Float32) bad(op, "dweights must be float32 of ids' shape");
  Array out = Array::empty(logits.shape(), logits.dtype());
  const mlxq_routing r = {(int32_t*)ids.data(), nullptr, nullptr, nullptr, ids.dim(0), ids.dim(1), logits.dim(1)};
  const mlxq_router o = {scoring, ids.dim(1), nullptr, 1, 1, 1, normalize, scale};
  check(mlxq_route_experts_backward((const float*)dweights.data(), logits.data(), dt, logits.dim(1), &o, &r, out.data(), s));
  return out;
}

void MxExperts::forward_into(const Mx& x, const Routing& r, bool combine, const Array& y, hipStream_t s) const {
  const char* op = "mx_experts";
  const mlxq_mx xv = view(x, op, "x"), wv = view(w, op, "w");
  if (w.codes.ndim() != 3 || w.K() != x.K()) bad(op, "w must be [experts, N, K] of x's K");
  const int64_t E = w.codes.dim(0), N = w.codes.dim(1);
  const mlxq_routing rv = routing_of(r, E, op);
  const bool per = x.codes.ndim() == 3;
  if ((x.codes.ndim() != 2 && !per) || x.codes.dim(0) != rv.tokens || (per && x.codes.dim(1) != rv.top_k))
    bad(op, "x must be [tokens, K] or [tokens, top_k, K]");
  if (y.shape() != (combine ? std::vector<int64_t>{rv.tokens, N} : std::vector<int64_t>{rv.tokens, rv.top_k, N})) bad(op, "y has another shape");
  int bdt;
  const void* b = bias_of(bias, {E, N}, op, bdt);
  const int ydt = abi_dtype(y.dtype(), op);
  const size_t need = mlxq_mx_experts_workspace_size(rv.tokens, rv.top_k, N, combine, ydt);
  const Array& ws = workspace_.at_least(need);
  check(mlxq_mx_experts(&xv, per, x.K(), &wv, N, b, bdt, &rv, combine, y.data(), ydt, ws.data(), ws.nbytes(), s));
}

Array MxExperts::forward(const Mx& x, const Routing& r, bool combine, hipStream_t s) const {
  if (w.codes.ndim() != 3 || r.ids.ndim() != 2) bad("mx_experts", "w must be [experts, N, K] and ids [tokens, top_k]");
  const int64_t T = r.ids.dim(0), k = r.ids.dim(1), N = w.codes.dim(1);
  Array y = Array::empty(combine ? std::vector<int64_t>{T, N} : std::vector<int64_t>{T, k, N}, out);
  forward_into(x, r, combine, y, s);
  return y;
}

}  // namespace mlxq
