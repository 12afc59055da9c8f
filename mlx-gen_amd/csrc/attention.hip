// attention.hip — how a paged attention call is cut up, and the join of split sequences.
#include <algorithm>

#include "paged.h"

namespace mlxq {

// One row's splits, joined by a workgroup.  The splits' sums are relative to their own maxima; each is weighted by
// exp2 of its maximum less the largest.  A thread takes 4 features of every (256 / (D / 4))-th split, so that a
// long sequence's splits are in flight together; the threads' sums are added in a fixed order.  Bound by latency: 56 rows
// of up to 196 splits of 128 features, 5.6 MB: 6.8 us.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int Hq) {
  __shared__ float weight[kMaxSplits], top_of[4], sum_of[4];
  __shared__ f32x4 add[256];
  const int tid = threadIdx.x, t = blockIdx.x / Hq, qh = blockIdx.x - t * Hq;
  const int from = min(max(a.batch.q_starts[0], 0), a.batch.T), to = min(a.batch.q_starts[a.batch.B], a.batch.T);
  if (t < from || t >= to) return;
  const int64_t row = blockIdx.x;
  const int ns = min(a.splits[row], a.S);
  if (ns <= 1) return;  // written by its one split
  f32x2 e = {-INFINITY, 0.0f};
  if (tid < ns) e = reinterpret_cast<const f32x2*>(a.ml)[row * a.S + tid];
  float top = e[0];
#pragma unroll
  for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
  if ((tid & 63) == 0) top_of[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
  const float ref = top == -INFINITY ? 0.0f : top, f = __builtin_amdgcn_exp2f(e[0] - ref);
  float l = e[1] * f;
  weight[tid] = f;
#pragma unroll
  for (int i = 32; i; i >>= 1) l += __shfl_xor(l, i);
  if ((tid & 63) == 0) sum_of[tid >> 6] = l;
  __syncthreads();
  const int per = a.D / 4, groups = 256 / per, gi = tid / per, d = (tid - gi * per) * 4;
  f32x4 v = {0, 0, 0, 0};
  if (gi < groups) {
    const float* p = a.part + row * a.S * a.D + d;
#pragma unroll 4
    for (int k = gi; k < ns; k += groups) v += *reinterpret_cast<const f32x4*>(p + (int64_t)k * a.D) * weight[k];
  }
  add[tid] = v;
  __syncthreads();
  if (tid >= per) return;
  for (int k = 1; k < groups; ++k) v += add[k * per + tid];
  l = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
  if (a.sinks) l += __builtin_amdgcn_exp2f(a.sinks[qh] * 1.44269504088896341f - ref);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* y = (T*)a.out.p + t * a.out.ts + qh * a.out.hs + d;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(y) = v * inv;
  else *reinterpret_cast<u32x2*>(y) = u32x2{Elem<T>::pack2(v[0] * inv, v[1] * inv), Elem<T>::pack2(v[2] * inv, v[3] * inv)};
}

// The same with a wave a row, for up to 64 splits: its lanes hold the splits' weights, 64 / (D / 4) groups of them the
// features.  Most rows of a step have one split only, and a quarter of the workgroups find that out sooner (48 sequences, 64
// heads of 64: 4.2 us).  8000 rows of four splits of 256 features, 37 MB: 8.2 us, 4.5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_rows_kernel(AttnArgs a, Divisor by_hq, int rows) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int t = by_hq.div(row), qh = row - t * (int)by_hq.d;
  const int from = min(max(a.batch.q_starts[0], 0), a.batch.T), to = min(a.batch.q_starts[a.batch.B], a.batch.T);
  if (t < from || t >= to) return;
  const int ns = min(a.splits[row], a.S);
  if (ns <= 1) return;  // written by its one split
  f32x2 e = {-INFINITY, 0.0f};
  if (lane < ns) e = reinterpret_cast<const f32x2*>(a.ml)[(int64_t)row * a.S + lane];
  const int per = a.D / 4, groups = 64 / per, gi = lane / per, d = (lane - gi * per) * 4;
  float top = e[0];
#pragma unroll
  for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
  const float ref = top == -INFINITY ? 0.0f : top, f = __builtin_amdgcn_exp2f(e[0] - ref);
  float l = e[1] * f;
#pragma unroll
  for (int i = 32; i; i >>= 1) l += __shfl_xor(l, i);
  f32x4 v = {0, 0, 0, 0};
  const float* p = a.part + (int64_t)row * a.S * a.D + d;
  for (int k0 = 0; k0 < ns; k0 += groups) {
    const int k = k0 + gi;
    const float w = __shfl(f, k & 63);
    if (gi < groups && k < ns) v += *reinterpret_cast<const f32x4*>(p + k * a.D) * w;
  }
  f32x4 all = v;
  for (int k = 1; k < groups; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) all[i] += __shfl(v[i], (lane + k * per) & 63);
  if (gi) return;
  if (a.sinks) l += __builtin_amdgcn_exp2f(a.sinks[qh] * 1.44269504088896341f - ref);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* y = (T*)a.out.p + t * a.out.ts + qh * a.out.hs + d;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(y) = all * inv;
  else *reinterpret_cast<u32x2*>(y) = u32x2{Elem<T>::pack2(all[0] * inv, all[1] * inv), Elem<T>::pack2(all[2] * inv, all[3] * inv)};
}

AttnPlan plan_attention(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype, int64_t B, int64_t max_q,
                        int64_t max_kv, int64_t window, bool causal) {
  AttnPlan p;
  const int64_t G = Hq / Hkv, cus = device_cu_count(), most = max_q * G;
  // Two row tiles a wave where they leave a SIMD two waves: not past 128 features, not in f32 (three prompts of up to
  // 900, 80-wide heads, in kernels of 128 features: 77.7 us with 32 rows, 56.2 with 16).
  p.rows = most <= 16 || D > 128 || dtype == MLXQ_FLOAT32 ? 16 : 32;
  p.tiled = dtype != MLXQ_FLOAT32 && most > p.rows;
  if (p.tiled) p.rows = 128;
  // Tiles of rows: at most one for every p.rows rows and a part one for every sequence.
  const int64_t tiles = T * G / p.rows + std::min(B, T);
  p.direct = !p.tiled && most <= p.rows;
  // Splits: enough workgroups of four waves for those that the CUs hold (tiled: two each, one for heads past 128) or
  // three on every CU, of at least 128 tokens (a unit for each wave: one token over 777, 8 heads: 9.5 us; 256: 10.1, one
  // split: 10.3) or 256 (tiled).  One row tile a sequence: of at most 768, since the sequences of a step are of unequal
  // length and the workgroups of a long one fill the chip more evenly (48 of up to 6000 tokens: 24.1 us, with 1024 25.3, with
  // 4096 39.3; one of 150001: 68.2, 71.7; 16 of up to 20000, most of them short: 44.9, with 8192 64.6).  Eight other shapes
  // in bf16 and fp16 are within 6 % of the best of 384 to 8192; f32 likes longer ones (12 of up to 9000: 50.9, with 2048 43.6).
  int64_t range = std::min<int64_t>(max_kv, 0x3fffff80);  // places end at 2^30
  // With a window a tile's rows see as many tokens as it holds and one for each of theirs, or, where they see all later
  // tokens, one for each of the step's, since the first row's window starts that far before the sequence's end (2000 tokens
  // over 16384, 8 heads of 128, window 128: 37.6 us, planned as causal 45.8; 300: 17.6 and 16.6).  How far a prefix
  // reaches is not known here: the last split takes what is past the plan.
  if (window) range = std::min(range, window + (causal ? std::min(max_q, p.rows / G + 1) : max_q));
  const int64_t slots = (!p.tiled ? 3 : D <= 128 ? 2 : 1) * cus, want = std::max<int64_t>(1, slots / std::max<int64_t>(tiles * Hkv, 1));
  auto whole = [&](int64_t n) { return p.tiled ? (n + 63) / 64 * 64 : (n + 127) / 128 * 128; };  // tiles; a unit a wave
  int64_t chunk = std::max<int64_t>(p.tiled ? 256 : 128, whole((range + want - 1) / want));
  // With many sequences and a long hint that is many workgroups and partial results: at most 16 for each that the chip
  // holds, and 256 MiB (which only more tokens than max_q promises reach).  256 sequences of up to 2000 tokens, 64 + 8
  // heads of 128, planned for 131072: 228 us and 55 MB, without the bound 835 and 1.46 GB, with 4 for each 224; one of them
  // of 131072 tokens: 600, 958 and 1215.
  if (p.direct) {
    const int64_t items = std::min(std::min(B, T) * Hkv, 16 * slots), most_splits = std::max<int64_t>(1, (256 << 20) / (T * Hq * D * 4));
    chunk = std::min<int64_t>(chunk, 768);
    chunk = std::max({chunk, whole((range * items + 16 * slots - 1) / (16 * slots)), whole((range + most_splits - 1) / most_splits)});
  }
  chunk = std::max(chunk, whole((range + kMaxSplits - 1) / kMaxSplits));
  p.chunk = (int)chunk;
  p.S = (int)std::max<int64_t>(1, (range + p.chunk - 1) / p.chunk);
  p.blocks = (p.direct ? B * p.S : p.tiled ? tiles : tiles * p.S) * Hkv;
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
  const int64_t rows = (int64_t)a.batch.T * a.Hkv * a.G;  // with splits, of 31 bits: see plan_attention's bounds
  // A wave's 64 lanes hold the weights of 64 splits; it sums those in turn that a workgroup sums in parallel.
  if (a.S <= 64)
    hipLaunchKernelGGL((attn_join_rows_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, Divisor(a.Hkv * a.G), (int)rows);
  else
    hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, st, a, a.Hkv * a.G);
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
