// workspace_test.cpp — the workspaces that the C++ host API keeps between calls, run by pytest.
//
//   workspace_test cpu   what is allocated and freed, counted by an allocator of this program's own
//   workspace_test gpu   a captured call replayed after a larger call on the same object
//
// Prints one line per case and exits non-zero if anything failed.
#include <dlfcn.h>

#include <cstdio>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include "../../include/mlxq.h"
#include "../../mlx-gen_amd/host/mlxq.hpp"

using namespace mlxq;

// In the cpu mode the host API's device memory is counted and never handed to a kernel: it starts 8 bytes off, where
// the library refuses it as a workspace, so that no call gets as far as a launch.
static bool g_count = false;
static int g_allocs = 0, g_frees = 0;
static size_t g_last = 0;

extern "C" hipError_t hipMalloc(void** p, size_t n) {
  if (!g_count) return ((hipError_t(*)(void**, size_t))dlsym(RTLD_NEXT, "hipMalloc"))(p, n);
  ++g_allocs;
  g_last = n;
  *p = (void*)(((uintptr_t)g_allocs << 40) + 8);
  return hipSuccess;
}
extern "C" hipError_t hipFree(void* p) {
  if (!g_count) return ((hipError_t(*)(void*))dlsym(RTLD_NEXT, "hipFree"))(p);
  ++g_frees;
  return hipSuccess;
}

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

static Array fake(std::vector<int64_t> s, Dtype d) { return Array::borrow((void*)4096, std::move(s), d); }

static void attention_cpu() {
  const auto shapes = cache_shapes(5000, 2, 16, 64, Dtype::Bfloat16);
  const Array k = fake(shapes.first, Dtype::Bfloat16), v = fake(shapes.second, Dtype::Bfloat16), q = fake({1, 4, 64}, Dtype::Bfloat16);
  // A step over max_kv tokens, refused for the workspace's alignment once it has one.
  auto call = [&](const PagedAttention& a, int64_t max_kv) {
    const CacheBatch b = {fake({1, 5000}, Dtype::Int32), fake({2}, Dtype::Int32), fake({1}, Dtype::Int32), 1, max_kv};
    bool refused = false;
    try {
      a.forward_into(q, k, v, b, q);
    } catch (const Error& e) {
      refused = e.status == MLXQ_EINVAL && strstr(e.what(), "workspace must be 16-byte aligned");
    }
    EXPECT(refused);
  };
  g_allocs = g_frees = 0;
  {
    banner("a larger call keeps the memory of a smaller one");
    PagedAttention a;
    call(a, 1000);
    EXPECT(g_allocs == 1);
    call(a, 1000);
    call(a, 900);
    EXPECT(g_allocs == 1);
    call(a, 60000);
    EXPECT(g_allocs == 2 && g_frees == 0);

    banner("a copy has memory of its own");
    const PagedAttention b = a;
    call(b, 1000);
    EXPECT(g_allocs == 3 && g_frees == 0);
    call(a, 60000);
    EXPECT(g_allocs == 3);

    banner("what is assigned to keeps its memory");
    PagedAttention c;
    call(c, 1000);
    EXPECT(g_allocs == 4);
    c = a;
    call(c, 1000);
    EXPECT(g_allocs == 4 && g_frees == 0);
    c = PagedAttention();
    EXPECT(g_frees == 0);
    call(c, 1000);
    EXPECT(g_allocs == 4);

    banner("what is moved from starts anew");
    PagedAttention e;
    e = std::move(c);
    call(e, 1000);
    EXPECT(g_allocs == 4);
    call(c, 1000);
    EXPECT(g_allocs == 5 && g_frees == 0);

    banner("slow growth allocates seldom");
    PagedAttention d;
    for (int64_t n = 1000; n < 60000; n += 100) call(d, n);
    EXPECT(g_allocs <= 5 + 7);
  }
  banner("all of it goes with the objects");
  EXPECT(g_frees == g_allocs);
}

// A refused call: its output or its workspace starts 8 bytes off.
template <typename F>
static void refused(F&& f) {
  bool yes = false;
  try {
    f();
  } catch (const Error& e) {
    yes = e.status == MLXQ_EINVAL && strstr(e.what(), "must be 16-byte aligned");
  }
  EXPECT(yes);
}

static void linear_cpu() {
  constexpr int64_t K = 256, N = 512, R = 16;
  const Dtype B = Dtype::Bfloat16;
  g_allocs = g_frees = 0;
  {
    banner("QuantizedLinear: more rows keep the memory of fewer, a copy has its own");
    const QuantizedLinear q{fake({N, K / 8}, Dtype::Uint32), fake({N, K / 64}, B), fake({N, K / 64}, B), std::nullopt, 64, 4};
    const Adapter lora = Adapter::lora(fake({K, R}, B), fake({R, N}, B), 1.0f);
    auto call = [&](const QuantizedLinear& l, int64_t M) {
      const Array out = fake({M, N}, B);
      refused([&] { l.forward_fused(fake({M, K}, B), &lora, MLXQ_ACT_NONE, nullptr, &out); });
    };
    call(q, 1);
    call(q, 1);
    EXPECT(g_allocs == 1);
    call(q, 4000);
    EXPECT(g_allocs == 2 && g_frees == 0);
    const QuantizedLinear r = q;
    call(r, 4000);
    EXPECT(g_allocs == 3 && g_frees == 0);
    call(q, 4000);
    EXPECT(g_allocs == 3);
  }
  EXPECT(g_frees == 3);
  g_allocs = g_frees = 0;
  {
    banner("AdaptableLinear: so does a partial sum that an f32 adapter follows");
    AdaptableLinear l = AdaptableLinear::from_quantized_parts(fake({N, K / 8}, Dtype::Uint32), fake({N, K / 64}, B), fake({N, K / 64}, B),
                                                              std::nullopt, 64, 4);
    l.push(Adapter::lora(fake({K, R}, B), fake({R, N}, B), 1.0f));
    l.push(Adapter::lora(fake({K, R}, Dtype::Float32), fake({R, N}, Dtype::Float32), 1.0f));
    auto call = [&](const AdaptableLinear& l, int64_t M) { refused([&] { l.forward_into(fake({M, K}, B), fake({M, N}, Dtype::Float32)); }); };
    call(l, 2);
    EXPECT(g_allocs == 2);  // the sum, and the base layer's workspace
    call(l, 4000);
    EXPECT(g_allocs == 4 && g_frees == 0);
    call(l, 2);
    call(l, 300);
    EXPECT(g_allocs == 4 && g_frees == 0);
    const AdaptableLinear c = l;
    call(c, 2);
    EXPECT(g_allocs == 6 && g_frees == 0);
  }
  EXPECT(g_frees == 6);
}

static Array upload(const std::vector<float>& v, std::vector<int64_t> shape) { return Array::from_host(v.data(), std::move(shape), Dtype::Float32); }
static Array upload(const std::vector<int32_t>& v, std::vector<int64_t> shape) { return Array::from_host(v.data(), std::move(shape), Dtype::Int32); }

static std::vector<float> host(const Array& a) {
  std::vector<float> v(a.size());
  a.to_host(v.data());
  return v;
}

static void attention_gpu() {
  banner("a captured step, a larger call, the step replayed");
  constexpr int64_t H = 2, D = 64, P = 16, PAGES = 400;
  std::mt19937 g(3);
  std::normal_distribution<float> nd;
  auto randn = [&](std::vector<int64_t> shape) {
    int64_t n = 1;
    for (int64_t d : shape) n *= d;
    std::vector<float> v(n);
    for (auto& x : v) x = nd(g);
    return upload(v, shape);
  };
  const auto shapes = cache_shapes(PAGES, H, P, D, Dtype::Float32);
  const Array k = randn(shapes.first), v = randn(shapes.second);
  std::vector<int32_t> row(PAGES);
  for (int i = 0; i < PAGES; ++i) row[i] = (7 * i + 3) % PAGES;
  const Array tables = upload(row, {1, PAGES});
  const CacheBatch small = {tables, upload(std::vector<int32_t>{0, 1}, {2}), upload(std::vector<int32_t>{1000}, {1}), 1, 1000};
  const CacheBatch large = {tables, upload(std::vector<int32_t>{0, 7}, {2}), upload(std::vector<int32_t>{6400}, {1}), 7, 6400};
  const Array q = randn({1, 2 * H, D}), wide = randn({7, 2 * H, D}), out = Array::empty(q.shape(), Dtype::Float32);
  const std::vector<float> want = host(PagedAttention().forward(q, k, v, small)), other = host(PagedAttention().forward(wide, k, v, large));

  const PagedAttention a;
  a.forward_into(q, k, v, small, out);
  hipStream_t s;
  hipGraph_t gr;
  hipGraphExec_t ex;
  EXPECT(hipStreamCreate(&s) == hipSuccess);
  EXPECT(hipDeviceSynchronize() == hipSuccess);
  EXPECT(hipStreamBeginCapture(s, hipStreamCaptureModeGlobal) == hipSuccess);
  a.forward_into(q, k, v, small, out, s);
  EXPECT(hipStreamEndCapture(s, &gr) == hipSuccess);
  EXPECT(hipGraphInstantiate(&ex, gr, nullptr, nullptr, 0) == hipSuccess);
  EXPECT(host(a.forward(wide, k, v, large)) == other);
  // Memory of many sizes: some of it would be what a freed workspace left.
  std::vector<Array> rest;
  for (int i = 0; i < 40; ++i) rest.push_back(upload(std::vector<float>(256 << (i % 10), 1.0f + i), {256 << (i % 10)}));
  for (int i = 0; i < 4; ++i) {
    EXPECT(hipMemset(out.data(), 0xff, out.nbytes()) == hipSuccess);
    EXPECT(hipDeviceSynchronize() == hipSuccess);
    EXPECT(hipGraphLaunch(ex, s) == hipSuccess);
    EXPECT(hipStreamSynchronize(s) == hipSuccess);
    EXPECT(host(out) == want);
    EXPECT(host(a.forward(wide, k, v, large)) == other);
  }
  for (int i = 0; i < 40; ++i) EXPECT(host(rest[i]) == std::vector<float>(256 << (i % 10), 1.0f + i));
  (void)hipGraphExecDestroy(ex);
  (void)hipGraphDestroy(gr);
  (void)hipStreamDestroy(s);
}

static void linear_gpu() {
  banner("a captured layer with two adapters, more rows, the layer replayed");
  constexpr int64_t K = 256, N = 512, R = 16, M = 4, MANY = 700;
  std::mt19937 g(5);
  std::normal_distribution<float> nd;
  auto randn = [&](std::vector<int64_t> shape, float std) {
    std::vector<float> v(shape[0] * shape[1]);
    for (auto& x : v) x = nd(g) * std;
    return upload(v, shape);
  };
  auto bf16 = [&](std::vector<int64_t> shape, float std) { return as_dtype(randn(shape, std), Dtype::Bfloat16); };
  const Packed p = quantize(bf16({N, K}, 0.05f), 64, 4);
  AdaptableLinear l = AdaptableLinear::from_quantized_parts(p.wq, p.scales, p.biases, std::nullopt, 64, 4);
  l.push(Adapter::lora(bf16({K, R}, 0.1f), bf16({R, N}, 0.1f), 0.5f));
  l.push(Adapter::lora(randn({K, R}, 0.1f), randn({R, N}, 0.1f), 1.25f));
  const Array x = bf16({M, K}, 1.0f), many = bf16({MANY, K}, 1.0f);
  const Array out = Array::empty({M, N}, Dtype::Float32);
  l.forward_into(x, out);
  const std::vector<float> want = host(out);
  hipStream_t s;
  hipGraph_t gr;
  hipGraphExec_t ex;
  EXPECT(hipStreamCreate(&s) == hipSuccess);
  EXPECT(hipDeviceSynchronize() == hipSuccess);
  EXPECT(hipStreamBeginCapture(s, hipStreamCaptureModeGlobal) == hipSuccess);
  l.forward_into(x, out, s);
  EXPECT(hipStreamEndCapture(s, &gr) == hipSuccess);
  EXPECT(hipGraphInstantiate(&ex, gr, nullptr, nullptr, 0) == hipSuccess);
  const Array wide = Array::empty({MANY, N}, Dtype::Float32);
  l.forward_into(many, wide);
  const std::vector<float> other = host(wide);
  std::vector<Array> rest;
  for (int i = 0; i < 40; ++i) rest.push_back(upload(std::vector<float>(256 << (i % 10), 1.0f + i), {256 << (i % 10)}));
  for (int i = 0; i < 4; ++i) {
    EXPECT(hipMemset(out.data(), 0xff, out.nbytes()) == hipSuccess);
    EXPECT(hipDeviceSynchronize() == hipSuccess);
    EXPECT(hipGraphLaunch(ex, s) == hipSuccess);
    EXPECT(hipStreamSynchronize(s) == hipSuccess);
    EXPECT(host(out) == want);
    l.forward_into(many, wide);
    EXPECT(host(wide) == other);
  }
  for (int i = 0; i < 40; ++i) EXPECT(host(rest[i]) == std::vector<float>(256 << (i % 10), 1.0f + i));
  (void)hipGraphExecDestroy(ex);
  (void)hipGraphDestroy(gr);
  (void)hipStreamDestroy(s);
}

int main(int argc, char** argv) {
  const std::string what = argc > 1 ? argv[1] : "cpu";
  try {
    g_count = what != "gpu";
    if (g_count) {
      attention_cpu();
      linear_cpu();
    } else {
      attention_gpu();
      linear_gpu();
    }
  } catch (const std::exception& e) {
    fprintf(stderr, "FAIL: %s\n", e.what());
    ++g_failures;
  }
  if (g_failures == 0) printf("ALL PASS\n");
  return g_failures != 0;
}
