// mx_matmul.hip — choice of the microscaled product's instances, and the weighted sum of the experts' products.
#include "mx.h"

namespace mlxq {

int run_mx_product_e4m3(const MxProduct& p, hipStream_t st);
int run_mx_product_e4m3_f32(const MxProduct& p, hipStream_t st);
int run_mx_product_e2m1(const MxProduct& p, hipStream_t st);

int run_mx_product(const MxProduct& p, int format, hipStream_t st) {
  if (format == kE2M1) return run_mx_product_e2m1(p, st);
  return p.y_dtype == MLXQ_BFLOAT16 ? run_mx_product_e4m3(p, st) : run_mx_product_e4m3_f32(p, st);
}

namespace {

// out[t, n] = sum_j w[t, j] y[t, j, n] over the choices with an expert, f32, rounded once.  The products y have out's type, as a
// caller's own sum would find them, at half of f32's bytes in the workspace and on the way: with bf16 the sum of four is off by 0.0024 of
// it (norms, 4090 tokens through 4 of 32 experts of 2880 x 2880) and with f32 products, rounded once, by 0.0017; a caller who wants
// those asks for an f32 result.  Bound by the reading of y: 4090 tokens, 4 experts, 2880 features in bf16 24 us, 4.9 TB/s, a large
// copy's rate.  A thread holds four features; rows of any N
// start at any element.
template <typename T>
__global__ __launch_bounds__(256) void mx_combine_kernel(const T* __restrict__ y, const int32_t* __restrict__ ids,
                                                         const float* __restrict__ weights, int k, int E, int N, int units,
                                                         int64_t first, int64_t total, T* __restrict__ out) {
  const int64_t u = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= total) return;
  const int64_t t = u / units;
  const int n = (int)(u - t * units) * 4, count = min(4, N - n);
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j = 0; j < k; ++j) {
    if ((unsigned)ids[t * k + j] >= (unsigned)E) continue;
    const float w = weights[t * k + j];
    const T* p = y + (t * k + j) * N + n;
    T v[4];
    if (count == 4) __builtin_memcpy(v, p, sizeof(v));
    else
      for (int i = 0; i < 4; ++i) v[i] = i < count ? p[i] : T(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = fmaf(w, Act<T>::ld(v, i), s[i]);
  }
  T r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) Act<T>::st(r, i, s[i]);
  T* o = out + t * N + n;
  if (count == 4) __builtin_memcpy(o, r, sizeof(r));
  else
    for (int i = 0; i < 4; ++i)
      if (i < count) o[i] = r[i];
}

template <typename T>
int combine(const void* y, const int32_t* ids, const float* weights, int64_t T_, int64_t k, int64_t E, int64_t N, void* out,
            hipStream_t st) {
  const int64_t units = (N + 3) / 4, total = T_ * units;
  return in_launches("mx_experts", (total + 255) / 256, 256, [&](int64_t group, unsigned grid) {
    mx_combine_kernel<T><<<grid, 256, 0, st>>>((const T*)y, ids, weights, (int)k, (int)E, (int)N, (int)units, group * 256, total, (T*)out);
  });
}

}  // namespace

int run_mx_combine(const void* y, int dtype, const int32_t* ids, const float* weights, int64_t T, int64_t k, int64_t E, int64_t N,
                   void* out, hipStream_t st) {
  if (dtype == MLXQ_BFLOAT16) return combine<uint16_t>(y, ids, weights, T, k, E, N, out, st);
  if (dtype == MLXQ_FLOAT16) return combine<_Float16>(y, ids, weights, T, k, E, N, out, st);
  return combine<float>(y, ids, weights, T, k, E, N, out, st);
}

}  // namespace mlxq
