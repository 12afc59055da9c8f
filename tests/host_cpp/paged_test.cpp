// paged_test.cpp — the paged-cache operators of the C++ host API, run by pytest.
//
//   paged_test cpu   shape checks and frequencies (no device work)
//   paged_test gpu   a prompt and steps of two sequences through append, attention and a fork, against the same
//                    in double precision here; forward_into captured in a HIP graph
//
// Prints one line per case and exits non-zero if anything failed.
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
  banner("frequencies");
  const RotaryFrequencies f = rotary_frequencies(64);
  EXPECT(f.inv_freq.size() == 32 && f.magnitude == 1.0 && f.inv_freq[0] == 1.0);
  EXPECT(std::fabs(f.inv_freq[31] - std::pow(10000.0, -62.0 / 64.0)) < 1e-18);
  EXPECT(rotary_frequencies(64, 1e4, MLXQ_ROPE_LINEAR, 4.0).inv_freq[0] == 0.25);
  EXPECT(status_of([] { rotary_frequencies(63); }) == MLXQ_EINVAL);
  EXPECT(status_of([] { rotary_frequencies(64, 1e4, 9); }) == MLXQ_EINVAL);
  banner("shape checks");
  auto fake = [](std::vector<int64_t> s, Dtype d) { return Array::borrow((void*)4096, std::move(s), d); };
  const auto shapes = cache_shapes(5, 2, 32, 64, Dtype::Bfloat16);
  EXPECT((shapes.first == std::vector<int64_t>{5, 2, 2, 8, 16, 8}) && (shapes.second == std::vector<int64_t>{5, 2, 4, 64, 8}));
  const Array k = fake(shapes.first, Dtype::Bfloat16), v = fake(shapes.second, Dtype::Bfloat16);
  const CacheBatch b = {fake({1, 4}, Dtype::Int32), fake({2}, Dtype::Int32), fake({1}, Dtype::Int32), 1, 64};
  const Array q = fake({3, 4, 64}, Dtype::Bfloat16);
  const PagedAttention att;
  EXPECT(status_of([&] { att.forward_into(fake({3, 4, 32}, Dtype::Bfloat16), k, v, b, q); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { att.forward_into(fake({3, 4, 64}, Dtype::Float32), k, v, b, q); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { att.forward_into(q, k, k, b, q); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { att.forward_into(q, k, v, b, fake({3, 2, 64}, Dtype::Bfloat16)); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { att.forward_into(fake({3, 3, 64}, Dtype::Bfloat16), k, v, b, fake({3, 3, 64}, Dtype::Bfloat16)); }) == MLXQ_EINVAL);
  PagedAttention bad_sinks;
  bad_sinks.sinks = fake({3}, Dtype::Float32);
  EXPECT(status_of([&] { bad_sinks.forward_into(q, k, v, b, fake({3, 4, 64}, Dtype::Bfloat16)); }) == MLXQ_EINVAL);
  CacheBatch short_lens = b;
  short_lens.kv_lens = fake({2}, Dtype::Int32);
  EXPECT(status_of([&] { att.forward_into(q, k, v, short_lens, q); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { cache_append(fake({3, 1, 64}, Dtype::Bfloat16), fake({3, 2, 64}, Dtype::Bfloat16), k, v, b); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { rotary(q, fake({2}, Dtype::Int32), fake({9, 32, 2}, Dtype::Float32)); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { copy_pages(k, 5, fake({1}, Dtype::Int32), fake({1}, Dtype::Int32)); }) == MLXQ_EINVAL);
  EXPECT(status_of([&] { copy_pages(k, 0, fake({2}, Dtype::Int32), fake({1}, Dtype::Int32)); }) == MLXQ_EINVAL);
}

// One sequence's tokens and the step's queries in f32; D features, H key heads, 2 H query heads.
constexpr int64_t H = 2, D = 32, P = 16;

static std::vector<float> randn(std::mt19937& g, size_t n) {
  std::normal_distribution<float> d;
  std::vector<float> v(n);
  for (auto& x : v) x = d(g);
  return v;
}
static Array upload(const std::vector<float>& v, std::vector<int64_t> shape) { return Array::from_host(v.data(), std::move(shape), Dtype::Float32); }
static Array upload(const std::vector<int32_t>& v, std::vector<int64_t> shape) { return Array::from_host(v.data(), std::move(shape), Dtype::Int32); }

static void turn(std::vector<double>& x, int64_t pos, const RotaryFrequencies& f) {
  for (int64_t h = 0; h < (int64_t)x.size() / D; ++h)
    for (int64_t i = 0; i < D / 2; ++i) {
      const double a = x[h * D + i], b = x[h * D + i + D / 2], c = std::cos(pos * f.inv_freq[i]), s = std::sin(pos * f.inv_freq[i]);
      x[h * D + i] = a * c - b * s;
      x[h * D + i + D / 2] = b * c + a * s;
    }
}

struct Tokens {
  std::vector<std::vector<double>> k, v;  // by token, [H * D]
};

// Row of query head h over the first n tokens.
static std::vector<double> attend(const std::vector<double>& q, const Tokens& t, int64_t n, int64_t h) {
  std::vector<double> z(n), o(D, 0.0);
  double top = -1e300, sum = 0.0;
  for (int64_t j = 0; j < n; ++j) {
    double s = 0.0;
    for (int64_t d = 0; d < D; ++d) s += q[h * D + d] * t.k[j][h / 2 * D + d];
    z[j] = s / std::sqrt((double)D);
    top = std::max(top, z[j]);
  }
  for (int64_t j = 0; j < n; ++j) sum += z[j] = std::exp(z[j] - top);
  for (int64_t j = 0; j < n; ++j)
    for (int64_t d = 0; d < D; ++d) o[d] += z[j] / sum * t.v[j][h / 2 * D + d];
  return o;
}

static void gpu() {
  std::mt19937 g(7);
  const RotaryFrequencies f = rotary_frequencies(D);
  const Array table = rotary_table(200, f);
  const int64_t pages = 12;
  const auto shapes = cache_shapes(pages, H, P, D, Dtype::Float32);
  const Array k_cache = Array::empty(shapes.first, Dtype::Float32), v_cache = Array::empty(shapes.second, Dtype::Float32);
  std::vector<std::vector<int32_t>> held = {{7, 2, 9}, {4}};
  std::vector<Tokens> book(2);
  const PagedAttention att;

  auto step = [&](const char* name, std::vector<int32_t> news, bool graph) {
    banner(name);
    const size_t B = book.size();
    int64_t T = 0, width = 0, max_q = 0, max_kv = 0;
    std::vector<int32_t> starts = {0}, lens;
    for (size_t b = 0; b < B; ++b) {
      T += news[b];
      starts.push_back((int32_t)T);
      lens.push_back((int32_t)book[b].k.size() + news[b]);
      width = std::max<int64_t>(width, held[b].size());
      max_q = std::max<int64_t>(max_q, news[b]);
      max_kv = std::max<int64_t>(max_kv, lens.back());
    }
    std::vector<int32_t> rows;
    for (size_t b = 0; b < B; ++b)
      for (int64_t i = 0; i < width; ++i) rows.push_back(i < (int64_t)held[b].size() ? held[b][i] : -1);
    const CacheBatch batch = {upload(rows, {(int64_t)B, width}), upload(starts, {(int64_t)B + 1}), upload(lens, {(int64_t)B}), max_q, max_kv};
    const std::vector<float> k = randn(g, T * H * D), v = randn(g, T * H * D), q = randn(g, T * 2 * H * D);
    const Array qa = upload(q, {T, 2 * H, D});
    const Array qr = cache_append(upload(k, {T, H, D}), upload(v, {T, H, D}), k_cache, v_cache, batch, &qa, &table);
    Array out = att.forward(qr, k_cache, v_cache, batch);
    if (graph) {
      hipStream_t s;
      hipGraph_t gr;
      hipGraphExec_t ex;
      EXPECT(hipStreamCreate(&s) == hipSuccess);
      EXPECT(hipDeviceSynchronize() == hipSuccess);
      EXPECT(hipStreamBeginCapture(s, hipStreamCaptureModeGlobal) == hipSuccess);
      att.forward_into(qr, k_cache, v_cache, batch, out, s);
      EXPECT(hipStreamEndCapture(s, &gr) == hipSuccess);
      EXPECT(hipGraphInstantiate(&ex, gr, nullptr, nullptr, 0) == hipSuccess);
      for (int i = 0; i < 3; ++i) {
        EXPECT(hipMemset(out.data(), 0xff, out.nbytes()) == hipSuccess);
        EXPECT(hipDeviceSynchronize() == hipSuccess);
        EXPECT(hipGraphLaunch(ex, s) == hipSuccess);
        EXPECT(hipStreamSynchronize(s) == hipSuccess);
      }
      (void)hipGraphExecDestroy(ex);
      (void)hipGraphDestroy(gr);
      (void)hipStreamDestroy(s);
    }
    std::vector<float> got(T * 2 * H * D);
    out.to_host(got.data());
    // f32 against double: scores of 32 terms and sums of up to 60 weights, all of order 1.  2^-24 (32 * 8 + 16 * 8 + 60) * 2
    // times values of at most 5 is 2.6e-4; a wrong token or feature is off by 0.1 and more.
    double worst = 0.0;
    int64_t t = 0;
    for (size_t b = 0; b < B; ++b)
      for (int32_t i = 0; i < news[b]; ++i, ++t) {
        const int64_t pos = (int64_t)book[b].k.size();
        std::vector<double> kt(k.begin() + t * H * D, k.begin() + (t + 1) * H * D), qt(q.begin() + t * 2 * H * D, q.begin() + (t + 1) * 2 * H * D);
        turn(kt, pos, f);
        turn(qt, pos, f);
        book[b].k.push_back(kt);
        book[b].v.emplace_back(v.begin() + t * H * D, v.begin() + (t + 1) * H * D);
        for (int64_t h = 0; h < 2 * H; ++h) {
          const std::vector<double> o = attend(qt, book[b], pos + 1, h);
          for (int64_t d = 0; d < D; ++d) worst = std::max(worst, std::fabs(o[d] - got[(t * 2 * H + h) * D + d]));
        }
      }
    printf("    worst error %.2e\n", worst);
    EXPECT(worst <= 2.6e-4);
  };

  step("prompts", {40, 5}, false);
  step("one token each", {1, 1}, true);
  banner("fork");
  held.push_back({7, 2, 11});  // shares the full pages, its own copy of the last
  book.push_back(book[0]);
  copy_pages(k_cache, 0, upload(std::vector<int32_t>{9}, {1}), upload(std::vector<int32_t>{11}, {1}));
  copy_pages(v_cache, 0, upload(std::vector<int32_t>{9}, {1}), upload(std::vector<int32_t>{11}, {1}));
  step("after the fork", {2, 1, 3}, true);
  banner("compaction moves a page and its entries");
  Array tables = upload(std::vector<int32_t>{7, 2, 11, 4}, {2, 2});
  const Array from = upload(std::vector<int32_t>{11}, {1}), to = upload(std::vector<int32_t>{0}, {1});
  copy_pages(k_cache, 0, from, to, &tables);
  copy_pages(v_cache, 0, from, to);
  std::vector<int32_t> rows(4);
  tables.to_host(rows.data());
  EXPECT((rows == std::vector<int32_t>{7, 2, 0, 4}));
  held[2][2] = 0;
  step("after the compaction", {1, 1, 1}, false);
}

int main(int argc, char** argv) {
  const std::string what = argc > 1 ? argv[1] : "cpu";
  try {
    if (what == "gpu") gpu();
    else cpu();
  } catch (const std::exception& e) {
    fprintf(stderr, "FAIL: %s\n", e.what());
    ++g_failures;
  }
  if (g_failures == 0) printf("ALL PASS\n");
  return g_failures != 0;
}
