// mx_test.cpp — the operators of a decoder block in microscaled types of the C++ host API, run by pytest.
//
//   mx_test cpu   shape checks (no device work)
//   mx_test gpu   a block: norm of a sum to 8 bits, a product, routing, experts, gradients, against the same in double
//                 precision here; forward_into captured in a HIP graph and replayed with other inputs
//
// Prints one line per case and exits non-zero if anything failed.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include "../../include/mlxq.h"
#include "../../mlx-gen_amd/host/mlxq.hpp"

using namespace mlxq;

static int g_failures = 0;
#define EXPECT(cond)                                              \
  do {                                                            \
    if (!(cond)) {                                                \
      fprintf(stderr, "FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      ++g_failures;                                               \
    }                                                             \
  } while (0)

static void banner(const char* name) {
  printf("[case] %s\n", name);
  fflush(stdout);
}

template <typename F>
static int status_of(F&& f) {
  try {
    f();
  } catch (const Error& e) {
    return e.status;
  }
  return MLXQ_OK;
}

static void cpu() {
  banner("shape checks");
  auto fake = [](std::vector<int64_t> s, Dtype d) { return Array::borrow((void*)4096, std::move(s), d); };
  const auto U8 = Dtype::Uint8, BF = Dtype::Bfloat16, F32 = Dtype::Float32, I32 = Dtype::Int32;
  const Mx x = {fake({3, 96}, U8), fake({3, 4}, U8), MLXQ_MX_E4M3}, w = {fake({5, 48}, U8), fake({5, 4}, U8), MLXQ_MX_E2M1};
  EXPECT(x.K() == 96 && w.K() == 96);
  EXPECT(status_of([&] { mx_quantize(fake({3, 40}, BF), MLXQ_MX_E2M1); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { mx_quantize(fake({3, 64}, BF), 7); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { mx_quantize(fake({3, 64}, I32), MLXQ_MX_E2M1); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { mx_dequantize({x.codes, fake({3, 3}, U8), MLXQ_MX_E4M3}); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { mx_dequantize({fake({3, 96}, F32), x.scales, MLXQ_MX_E4M3}); }) == MLXQ_EINVAL);
  MxLinear lin;
  lin.w = w;
  EXPECT(status_of([&] { lin.forward_into(x, fake({3, 6}, BF)); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { lin.forward_into({fake({3, 64}, U8), fake({3, 4}, U8), MLXQ_MX_E4M3}, fake({3, 5}, BF)); }) == MLXQ_EINVAL);
  lin.bias = fake({4}, BF);
  EXPECT(status_of([&] { lin.forward_into(x, fake({3, 5}, BF)); }) == MLXQ_EINVAL);
  lin.bias.reset();
  lin.w.format = MLXQ_MX_E4M3;
  lin.w = {fake({5, 96}, U8), fake({5, 4}, U8), MLXQ_MX_E4M3};
  EXPECT(status_of([&] { lin.forward_into(x, fake({3, 5}, BF)); }) == MLXQ_EUNSUPPORTED);
  const Array h = fake({3, 64}, BF), odd = fake({63}, BF), other = fake({3, 64}, F32);
  EXPECT(status_of([&] { rms_norm(h, &odd); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { rms_norm(h, nullptr, &other); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { rms_norm(fake({3, 40}, BF), nullptr, nullptr, 1e-6f, true); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { RmsNormGradient().backward(other, h); }) == MLXQ_EINVAL);
  Router router;
  EXPECT(status_of([&] { router.forward(fake({3}, BF)); }) == MLXQ_EINVAL);
  router.top_k = 0;
  EXPECT(status_of([&] { router.forward(fake({3, 8}, BF)); }) == MLXQ_EINVAL);
  router.top_k = 2;
  const Array act = fake({3}, U8);
  EXPECT(status_of([&] { router.forward(fake({3, 8}, BF), &act); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { router.backward(fake({3, 1}, F32), fake({3, 8}, BF), fake({3, 2}, I32)); }) == MLXQ_EINVAL);
  MxExperts ex;
  ex.w = {fake({4, 5, 48}, U8), fake({4, 5, 4}, U8), MLXQ_MX_E2M1};
  const Routing r = {fake({3, 2}, I32), fake({3, 2}, F32), fake({5}, I32), fake({6}, I32)};
  EXPECT(status_of([&] { ex.forward_into(x, r, false, fake({3, 5}, BF)); }) == MLXQ_EINVAL);
  Routing short_rows = r;
  short_rows.rows = fake({5}, I32);
  EXPECT(status_of([&] { ex.forward_into(x, short_rows, false, fake({3, 2, 5}, BF)); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { ex.forward_into({fake({4, 96}, U8), fake({4, 4}, U8), MLXQ_MX_E4M3}, r, false, fake({3, 2, 5}, BF)); }) == MLXQ_EINVAL);
}

static std::vector<float> randn(std::mt19937& g, size_t n, float std = 1.0f) {
  std::normal_distribution<float> d(0.0f, std);
  std::vector<float> v(n);
  for (auto& x : v) x = d(g);
  return v;
}
static Array up(const std::vector<float>& v, std::vector<int64_t> shape) { return Array::from_host(v.data(), std::move(shape), Dtype::Float32); }
template <typename T>
static std::vector<T> down(const Array& a) {
  std::vector<T> v(a.size());
  (void)hipDeviceSynchronize();
  if (!v.empty()) a.to_host(v.data());
  return v;
}

constexpr int64_t T = 9, K = 160, N = 40, E = 6, TOP = 2;

// What a microscaled array stands for, by the library's own dequantisation (checked against its definition elsewhere).
static std::vector<float> values(const Mx& x) { return down<float>(mx_dequantize(x, Dtype::Float32)); }

static bool near(const std::vector<float>& got, const std::vector<double>& want, const std::vector<double>& mag, double rel) {
  for (size_t i = 0; i < got.size(); ++i)
    if (!(std::fabs(got[i] - want[i]) <= rel * mag[i] + 1e-30)) return false;
  return got.size() == want.size();
}

static void gpu() {
  std::mt19937 g(5);
  const std::vector<float> xs = randn(g, T * K), rs = randn(g, T * K), ws = randn(g, K, 0.2f);
  const Array x = up(xs, {T, K}), res = up(rs, {T, K}), w = up(ws, {K});
  hipStream_t st;
  EXPECT(hipStreamCreate(&st) == hipSuccess);

  banner("norm of a sum");
  const Normed plain = rms_norm(x, &w, &res, 1e-5f, false, st), eight = rms_norm(x, &w, &res, 1e-5f, true, st);
  std::vector<double> want(T * K), mag(T * K);
  const std::vector<float> h = down<float>(plain.sum);
  for (int64_t t = 0; t < T; ++t) {
    double s = 0;
    for (int64_t k = 0; k < K; ++k) s += (double)h[t * K + k] * h[t * K + k];
    for (int64_t k = 0; k < K; ++k) {
      EXPECT(h[t * K + k] == xs[t * K + k] + rs[t * K + k]);
      want[t * K + k] = h[t * K + k] / std::sqrt(s / K + 1e-5) * ws[k];
      mag[t * K + k] = std::fabs(want[t * K + k]);
    }
  }
  EXPECT(near(down<float>(plain.y), want, mag, 96 * std::pow(2.0, -24)));
  // an 8-bit value is off by at most half a step, 2^-4 of it, or half the smallest step of its block, 2^-10 of 2^e <= max / 224
  const std::vector<float> v8 = values(eight.mx);
  for (int64_t i = 0; i < T * K; ++i) {
    double top = 0;
    for (int64_t k = i / 32 * 32; k < i / 32 * 32 + 32; ++k) top = std::max(top, mag[k]);
    EXPECT(std::fabs(v8[i] - want[i]) <= mag[i] / 16 + top / 224 / 1024);
  }

  banner("product");
  MxLinear lin;
  lin.w = mx_quantize(up(randn(g, N * K), {N, K}), MLXQ_MX_E2M1, st);
  lin.bias = up(randn(g, N), {N});
  lin.out = Dtype::Float32;
  const std::vector<float> wv = values(lin.w), bv = down<float>(*lin.bias);
  auto product = [&](const std::vector<float>& a, const float* weights, const float* b, std::vector<double>& y, std::vector<double>& m, int64_t row,
                     int64_t at) {
    for (int64_t n = 0; n < N; ++n) {
      double s = b[n], sm = std::fabs(b[n]);
      for (int64_t k = 0; k < K; ++k) {
        const double p = (double)a[row * K + k] * weights[n * K + k];
        s += p;
        sm += std::fabs(p);
      }
      y[at * N + n] = s;
      m[at * N + n] = sm;
    }
  };
  std::vector<double> y(T * N), ym(T * N);
  for (int64_t t = 0; t < T; ++t) product(v8, wv.data(), bv.data(), y, ym, t, t);
  const double f32_sum = (K / 32 + 18) * std::pow(2.0, -23);
  EXPECT(near(down<float>(lin.forward(eight.mx, st)), y, ym, f32_sum));

  banner("routing and experts");
  Router router;
  router.top_k = TOP;
  const std::vector<float> zs = randn(g, T * E);
  const Routing r = router.forward(up(zs, {T, E}), nullptr, st);
  const std::vector<int32_t> ids = down<int32_t>(r.ids), starts = down<int32_t>(r.starts), rows = down<int32_t>(r.rows);
  const std::vector<float> wt = down<float>(r.weights);
  for (int64_t t = 0; t < T; ++t) {
    std::vector<int> order(E);
    for (int e = 0; e < E; ++e) order[e] = e;
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return zs[t * E + a] > zs[t * E + b]; });
    double total = 0;
    for (int j = 0; j < TOP; ++j) total += std::exp((double)zs[t * E + order[j]]);
    for (int j = 0; j < TOP; ++j) {
      EXPECT(ids[t * TOP + j] == order[j]);
      EXPECT(std::fabs(wt[t * TOP + j] - std::exp((double)zs[t * E + order[j]]) / total) < 1e-7);
    }
  }
  EXPECT(starts[0] == 0 && starts[E] == T * TOP);
  for (int e = 0; e < E; ++e)
    for (int p = starts[e]; p < starts[e + 1]; ++p) EXPECT(ids[rows[p]] == e && (p == starts[e] || rows[p - 1] < rows[p]));
  const Routing again = router.plan(r.ids, r.weights, E, st);
  EXPECT(down<int32_t>(again.rows) == rows && down<int32_t>(again.starts) == starts);
  MxExperts ex;
  ex.w = mx_quantize(up(randn(g, E * N * K), {E, N, K}), MLXQ_MX_E2M1, st);
  ex.bias = up(randn(g, E * N), {E, N});
  ex.out = Dtype::Float32;
  const std::vector<float> ev = values(ex.w), eb = down<float>(*ex.bias);
  std::vector<double> each(T * TOP * N), em(T * TOP * N), sum(T * N, 0.0), sm(T * N, 0.0);
  for (int64_t c = 0; c < T * TOP; ++c) {
    product(v8, ev.data() + ids[c] * N * K, eb.data() + ids[c] * N, each, em, c / TOP, c);
    for (int64_t n = 0; n < N; ++n) {
      sum[c / TOP * N + n] += wt[c] * each[c * N + n];
      sm[c / TOP * N + n] += wt[c] * em[c * N + n];
    }
  }
  EXPECT(near(down<float>(ex.forward(eight.mx, r, false, st)), each, em, f32_sum));
  EXPECT(near(down<float>(ex.forward(eight.mx, r, true, st)), sum, sm, f32_sum + 4 * std::pow(2.0, -23)));

  banner("gradients");
  const std::vector<float> dys = randn(g, T * K), dws = randn(g, T * TOP);
  const auto grad = RmsNormGradient{1e-5f}.backward(up(dys, {T, K}), plain.sum, &w, &res, st);
  std::vector<double> dx(T * K), dxm(T * K), dw(K, 0.0), dwm(K, 0.0);
  for (int64_t t = 0; t < T; ++t) {
    double s = 0, gx = 0, gm = 0;
    for (int64_t k = 0; k < K; ++k) s += (double)h[t * K + k] * h[t * K + k];
    const double rr = 1 / std::sqrt(s / K + 1e-5);
    for (int64_t k = 0; k < K; ++k) {
      gx += (double)dys[t * K + k] * ws[k] * h[t * K + k];
      gm += std::fabs((double)dys[t * K + k] * ws[k] * h[t * K + k]);
    }
    for (int64_t k = 0; k < K; ++k) {
      const int64_t i = t * K + k;
      const double gv = (double)dys[i] * ws[k];
      dx[i] = rr * gv - rr * rr * rr * h[i] * gx / K + rs[i];
      dxm[i] = std::fabs(rr * gv) + rr * rr * rr * std::fabs(h[i]) * gm / K + std::fabs(rs[i]);
      dw[k] += dys[i] * h[i] * rr;
      dwm[k] += std::fabs(dys[i] * h[i] * rr);
    }
  }
  EXPECT(near(down<float>(grad.first), dx, dxm, 300 * std::pow(2.0, -24)));
  EXPECT(near(down<float>(grad.second), dw, dwm, 210 * std::pow(2.0, -24)));
  const std::vector<float> dz = down<float>(router.backward(up(dws, {T, TOP}), up(zs, {T, E}), r.ids, st));
  for (int64_t t = 0; t < T; ++t) {
    double mean = 0, m = 0;
    for (int j = 0; j < TOP; ++j) {
      mean += dws[t * TOP + j] * wt[t * TOP + j];
      m += std::fabs(dws[t * TOP + j]);
    }
    for (int e = 0; e < E; ++e) {
      double want_z = 0;
      for (int j = 0; j < TOP; ++j)
        if (ids[t * TOP + j] == e) want_z = wt[t * TOP + j] * (dws[t * TOP + j] - mean);
      EXPECT(std::fabs(dz[t * E + e] - want_z) <= 64 * std::pow(2.0, -24) * m);
    }
  }

  banner("graph");
  const Array out = Array::empty({T, N}, Dtype::Float32), sum_out = Array::empty({T, N}, Dtype::Float32);
  lin.forward_into(eight.mx, out, st);
  ex.forward_into(eight.mx, r, true, sum_out, st);  // its workspace is there from now on
  EXPECT(hipStreamSynchronize(st) == hipSuccess);
  hipGraph_t graph;
  hipGraphExec_t exec;
  EXPECT(hipStreamBeginCapture(st, hipStreamCaptureModeGlobal) == hipSuccess);
  lin.forward_into(eight.mx, out, st);
  ex.forward_into(eight.mx, r, true, sum_out, st);
  EXPECT(hipStreamEndCapture(st, &graph) == hipSuccess);
  EXPECT(hipGraphInstantiate(&exec, graph, nullptr, nullptr, 0) == hipSuccess);
  for (int turn = 0; turn < 3; ++turn) {
    const Mx fresh = mx_quantize(up(randn(g, T * K), {T, K}), MLXQ_MX_E4M3, st);
    EXPECT(hipMemcpyAsync(eight.mx.codes.data(), fresh.codes.data(), fresh.codes.nbytes(), hipMemcpyDeviceToDevice, st) == hipSuccess);
    EXPECT(hipMemcpyAsync(eight.mx.scales.data(), fresh.scales.data(), fresh.scales.nbytes(), hipMemcpyDeviceToDevice, st) == hipSuccess);
    const std::vector<float> eager = down<float>(lin.forward(fresh, st)), eager_sum = down<float>(ex.forward(fresh, r, true, st));
    EXPECT(hipGraphLaunch(exec, st) == hipSuccess);
    EXPECT(down<float>(out) == eager && down<float>(sum_out) == eager_sum);
  }
  EXPECT(hipGraphExecDestroy(exec) == hipSuccess && hipGraphDestroy(graph) == hipSuccess);
  EXPECT(hipStreamDestroy(st) == hipSuccess);
}

int main(int argc, char** argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  try {
    if (what == "cpu") cpu();
    else if (what == "gpu") gpu();
    else return 2;
  } catch (const Error& e) {
    fprintf(stderr, "FAIL: mlxq::Error(%d): %s\n", e.status, e.what());
    ++g_failures;
  }
  if (g_failures == 0) printf("ALL PASS\n");
  return g_failures != 0;
}
