// attention.hip — how a paged attention call is cut up, and the join of split sequences.
#include <algorithm>

#include "paged.h"

namespace mlxq {

// One row's splits, joined: thread (row, 4 features).  The splits' sums are relative to their own
// maxima; each is weighted by exp2 of its maximum less the largest, in the order of the splits.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int Hq, int64_t total) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int per = a.D / 4;
  const int64_t row = id / per, t = row / Hq;
  const int d = (int)(id - row * per) * 4, qh = (int)(row - t * Hq);
  const int from = min(max(a.batch.q_starts[0], 0), a.batch.T), to = min(a.batch.q_starts[a.batch.B], a.batch.T);
  if (t < from || t >= to) return;
  const int ns = min(a.splits[row], a.S);
  if (ns <= 1) return;  // written by its one split
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.ml) + row * a.S;
  float top = -INFINITY;
  for (int k = 0; k < ns; ++k) top = fmaxf(top, ml[k][0]);
  const float ref = top == -INFINITY ? 0.0f : top;
  f32x4 v = {0, 0, 0, 0};
  float l = 0.0f;
  for (int k = 0; k < ns; ++k) {
    const f32x2 e = ml[k];
    const float f = __builtin_amdgcn_exp2f(e[0] - ref);
    l += e[1] * f;
    v += *reinterpret_cast<const f32x4*>(a.part + (row * a.S + k) * a.D + d) * f;
  }
  if (a.sinks) l += __builtin_amdgcn_exp2f(a.sinks[qh] * 1.44269504088896341f - ref);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* y = (T*)a.out.p + t * a.out.ts + qh * a.out.hs + d;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(y) = v * inv;
  else *reinterpret_cast<u32x2*>(y) = u32x2{Elem<T>::pack2(v[0] * inv, v[1] * inv), Elem<T>::pack2(v[2] * inv, v[3] * inv)};
}

AttnPlan plan_attention(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype, int64_t B, int64_t max_q,
                        int64_t max_kv, int64_t window) {
  AttnPlan p;
  const int64_t G = Hq / Hkv, cus = device_cu_count(), most = max_q * G;
  // 32 rows of heads wider than 128 would not fit a wave's registers in the streaming kernel.
  p.rows = most <= 16 || D > 128 ? 16 : 32;
  p.tiled = dtype != MLXQ_FLOAT32 && most > p.rows;
  if (p.tiled) p.rows = 128;
  p.direct = !p.tiled && most <= p.rows;
  p.units = p.direct ? B : T * G / p.rows + B;
  // Splits: enough workgroups of four waves for two (tiled) or three on every CU, at least 256 tokens each.
  int64_t range = max_kv;
  if (window) range = std::min(range, window + max_q);
  const int64_t busy = std::min<int64_t>(p.units, T * G / p.rows + std::min(B, T)) * Hkv;
  const int64_t want = std::max<int64_t>(1, (p.tiled ? 2 : 3) * cus / std::max<int64_t>(busy, 1));
  int64_t chunk = std::max<int64_t>(256, (range + want - 1) / want);
  chunk = std::max<int64_t>((chunk + 127) / 128 * 128, ((range + 255) / 256 + 127) / 128 * 128);
  chunk = std::min<int64_t>(chunk, 0x40000000);
  p.chunk = (int)chunk;
  p.S = (int)std::max<int64_t>(1, (range + chunk - 1) / chunk);
  if (p.S > 1) {
    auto align = [](size_t b) { return (b + 255) / 256 * 256; };
    const size_t rows = (size_t)(T * Hq);
    p.ml = align(rows * p.S * D * 4);
    p.splits = p.ml + align(rows * p.S * 8);
    p.total = p.splits + align(rows * 4);
  }
  return p;
}

template <typename T>
static int launch_join(const AttnArgs& a, hipStream_t st) {
  const int64_t total = (int64_t)a.batch.T * a.Hkv * a.G * (a.D / 4), blocks = (total + 255) / 256;
  if (blocks > 0x7fffffff) return set_error(MLXQ_EINVAL, "paged_attention: problem too large");
  hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, st, a, a.Hkv * a.G, total);
  return check_launch("paged_attention");
}

int run_attention(const AttnArgs& a, int dtype, const AttnPlan& plan, hipStream_t st) {
  const int rc = dtype == MLXQ_BFLOAT16 ? (plan.tiled ? run_attn_tile_bf16 : run_attn_stream_bf16)(a, plan, st)
                 : dtype == MLXQ_FLOAT16 ? (plan.tiled ? run_attn_tile_f16 : run_attn_stream_f16)(a, plan, st)
                                         : run_attn_stream_f32(a, plan, st);
  if (rc || a.S == 1) return rc;
  if (dtype == MLXQ_BFLOAT16) return launch_join<uint16_t>(a, st);
  if (dtype == MLXQ_FLOAT16) return launch_join<_Float16>(a, st);
  return launch_join<float>(a, st);
}

}  // namespace mlxq
