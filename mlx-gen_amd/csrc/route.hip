// route.hip — routing of tokens to experts, the plan of the experts' products, and the gradient of the weights.
//
// A wave a token; expert e lies in lane e % 64, place e / 64.  Scores are compared as integers whose order is that of
// the numbers: the logits' own bits where there is no bias (f32: exact, and as the scores' order), else s + bias in 64
// bits.  top_k rounds of a maximum over the wave; ballots then find the lowest expert that has it.  A few loads and a few
// hundred instructions a token: a short call is a launch's latency, a long one bound by the vector units (17 tokens, 8 of 128
// experts in groups, f32 logits with a bias 6.5 us; 16381 tokens, 8 of 256 experts 26.5 us with the plan).  A second kernel makes
// the plan: with a wave a token and the plan in one workgroup, a launch less, 8 tokens took 9.3 us for 10.5, but 17 12.3 for 10.6.
//
// The plan is a stable counting sort of the choices by expert: segments count their experts, and each choice's place is
// its expert's start, plus that expert's choices in earlier segments and in earlier waves of its own, plus its rank in its
// wave; the rank among 64 is found by ballots, so that no result depends on the order of an atomic.
#include <algorithm>

#include "mx.h"

namespace mlxq {

namespace {

// Integers in the order of the numbers, above those for NaN (1) and for what is not to be chosen (0).
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 1;
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 as 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(double v) {
  if (v != v) return 1;
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}

template <typename V>
__device__ __forceinline__ V wave_max(V v) {
  return lanes_reduce(v, [](V a, V b) { return a > b ? a : b; });  // of floats: a NaN is passed over, or stays
}
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
  return lanes_reduce(v, [](V a, V b) { return a + b; });
}

// The largest of the wave's keys, and the lanes that hold it.  64-bit keys mostly differ in their upper halves.
__device__ __forceinline__ uint32_t wave_top(uint32_t k, unsigned long long& lanes) {
  const uint32_t m = wave_max(k);
  lanes = __ballot(k == m);
  return m;
}
__device__ __forceinline__ unsigned long long wave_top(unsigned long long k, unsigned long long& lanes) {
  const uint32_t hi = wave_max((uint32_t)(k >> 32));
  lanes = __ballot((uint32_t)(k >> 32) == hi);
  if ((lanes & (lanes - 1)) == 0) return (unsigned long long)hi << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, __builtin_ctzll(lanes));
  const uint32_t lo = wave_max((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  const unsigned long long m = (unsigned long long)hi << 32 | lo;
  lanes = __ballot(k == m);
  return m;
}

// WIDE: the choice is by s + bias, or a group's score is a sum: scores in 64 bits.
template <typename T, int NE, bool WIDE>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
  using Key = typename std::conditional<WIDE, unsigned long long, uint32_t>::type;
  using Val = typename std::conditional<WIDE, double, float>::type;
  __shared__ Val of_group[WIDE || NE > 0 ? 4 : 1][NE * 64];  // a wave's scores, for its groups
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = a.E;
  const int t = blockIdx.x * 4 + wave;
  if (t >= a.T) return;  // whole waves; no barrier below
  float z[NE];
  const T* row = (const T*)a.logits + t * a.row_stride;
#pragma unroll
  for (int i = 0; i < NE; ++i) z[i] = i * 64 + lane < E ? Act<T>::ld(row, i * 64 + lane) : -INFINITY;
  if (a.active && !a.active[t]) {
    if (lane < a.k) {
      a.ids[(int64_t)t * a.k + lane] = -1;
      a.weights[(int64_t)t * a.k + lane] = 0.0f;
    }
    return;
  }
  const bool soft = a.scoring == MLXQ_ROUTE_SOFTMAX;
  float top = -INFINITY;
  bool undefined = false;  // softmax of a row with NaN or +infinity
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    top = fmaxf(top, z[i]);
    undefined |= z[i] != z[i] || z[i] == INFINITY;
  }
  double total = 0.0, top64 = 0.0;
  if (soft) {
    top = wave_max(top);
    undefined = __any(undefined);
    top64 = top == -INFINITY ? 0.0 : (double)top;  // no expert is wanted: all scores 0
    if (WIDE || !a.normalize) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < NE; ++i) sum += i * 64 + lane < E ? exp((double)z[i] - top64) : 0.0;
      total = wave_sum(sum);
    }
  }
  auto score = [&](float v) {  // in 64 bits; softmax without its denominator where that cancels
    if (!soft) return 1.0 / (1.0 + exp(-(double)v));
    const double e = exp((double)v - top64);
    return WIDE || !a.normalize ? (total > 0.0 ? e / total : 0.0) : e;
  };
  // A softmax's row with NaN or +infinity has no scores: the choice goes by its logits alone, without the bias and a group by its
  // best, so that NaN still comes last.
  const bool alone = soft && undefined;
  Val val[NE];
  Key key[NE];
  double own[WIDE ? NE : 1];  // scores
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = i * 64 + lane;
    if constexpr (WIDE) {
      // A group's score without a bias is of scores; the choice then goes by the logits, whose order is theirs.
      val[i] = own[i] = e < E ? score(z[i]) : 0.0;
      if (a.bias) val[i] += e < E ? (double)a.bias[e] : 0.0;
      if (alone) val[i] = z[i];
      key[i] = e < E ? a.bias ? key_of(val[i]) : (Key)key_of(z[i]) : 0;
    } else {
      val[i] = z[i];
      key[i] = e < E ? key_of(z[i]) : 0;
    }
  }
  if (a.kept < a.groups) {
    // Lane g scores group g: its best, or the sum of its two best.  NaN counts as -infinity here.
    const int size = E / a.groups;
    Val* mine = of_group[wave];
#pragma unroll
    for (int i = 0; i < NE; ++i) mine[i * 64 + lane] = val[i];
    __builtin_amdgcn_wave_barrier();
    Val best = -INFINITY, next = -INFINITY;
    if (lane < a.groups)
      for (int e0 = 0; e0 < size; e0 += 8) {
        Val v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = mine[lane * size + min(e0 + e, size - 1)];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Val x = e0 + e < size ? v[e] : -INFINITY;
          const Val low = x > best ? best : x;  // of a NaN both comparisons fail
          if (x > best) best = x;
          if (low > next) next = low;
        }
      }
    Key gk = lane < a.groups ? key_of(a.best > 1 && size > 1 && !alone ? best + next : best) : 0;
    unsigned long long kept = 0;
    for (int j = 0; j < a.kept; ++j) {
      unsigned long long lanes;
      wave_top(gk, lanes);
      const int g = __builtin_ctzll(lanes);
      kept |= 1ull << g;
      if (lane == g) gk = 0;
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = i * 64 + lane;
      if (e < E && !(kept >> (e / size) & 1)) key[i] = 0;
    }
  }
  int id = 0;  // lane j < k: the j-th choice, and its logit or score
  float zj = 0.0f;
  double wj = 0.0;
  for (int j = 0; j < a.k; ++j) {
    Key m = key[0];
#pragma unroll
    for (int i = 1; i < NE; ++i) m = max(m, key[i]);
    unsigned long long lanes;
    m = wave_top(m, lanes);
    // Expert i * 64 + lane: the lowest has the lowest i, then the lowest lane.
    bool found = false;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const unsigned long long has = NE == 1 ? lanes : __ballot(key[i] == m);
      if (!found && has) {
        const int l = __builtin_ctzll(has);
        found = true;
        if (lane == l) key[i] = 0;
        if constexpr (WIDE) {
          const double v = lane_value(own[i], l);
          if (lane == j) wj = v;
        } else {
          const float v = lane_value(z[i], l);
          if (lane == j) zj = v;
        }
        if (lane == j) id = i * 64 + l;
      }
    }
  }
  double w = 0.0;
  if (lane < a.k) {
    if constexpr (WIDE) w = wj;
    else w = score(zj);
  }
  if (a.normalize) {
    const double sum = wave_sum(w);
    w = sum == 0.0 ? 0.0 : w / sum;
  }
  if (soft && undefined) w = __longlong_as_double(0x7ff8000000000000ll);
  if (lane < a.k) {
    a.ids[(int64_t)t * a.k + lane] = id;
    a.weights[(int64_t)t * a.k + lane] = (float)(w * (double)a.scale);
  }
}

// exp of x <= 0, correct to f32: the rounding of the product with log2 e is added back.
__device__ __forceinline__ float exp_of(float x) {
  const float t = x * 1.44269504088896341f, lost = fmaf(x, 1.44269504088896341f, -t) + x * 1.925963033500e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return e > 0.0f ? fmaf(e, lost * 0.693147180559945f, e) : e;  // -infinity: 0, and lost is no number
}

// dz from dw, with s the scores of a token and w = scale s / (their sum over the chosen, or 1), d = scale dw:
//   not normalized: softmax dz = s (d - sum d s), d being 0 for experts that were not chosen; sigmoid dz = d s (1 - s)
//   normalized: the chosen experts alone, with their shares v = s / (sum of s): dz = v (d - sum d v), times 1 - s of a sigmoid
// Lane j < k works out its choice; logits and results change lanes in LDS.
//
// Shares are ordinary numbers where scores leave f32's range (experts chosen by a bias, some 87 below the row's largest logit or
// below 0), so the exponentials are taken relative to the largest chosen logit: a sigmoid of z < 0 is exp(z) (1 - s).  Where the
// weights' scores are all 0 in the router's 64 bits, so are weights and gradient.
//
// A wave a token, whose loads, reductions and changes of lanes follow one another: 16381 tokens, 8 of 256 experts, bf16 7.9 us
// normalized (through the softmax of all experts 8.8), 8.3 not.
template <typename T, int NE>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteArgs a, const float* __restrict__ dweights, T* __restrict__ dz) {
  __shared__ float swap[4][NE * 64];
  const int lane = threadIdx.x & 63, E = a.E;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;  // whole waves; no barrier below
  float* mine = swap[threadIdx.x >> 6];
  float z[NE];  // of a softmax without normalization later the scores
  const T* row = (const T*)a.logits + t * a.row_stride;
#pragma unroll
  for (int i = 0; i < NE; ++i) z[i] = Act<T>::ld(row, min(i * 64 + lane, E - 1));
  const int64_t at = (int64_t)t * a.k + min(lane, a.k - 1);
  const int id = a.ids[at];
  float up = dweights[at] * a.scale;
  const bool chosen = lane < a.k && (unsigned)id < (unsigned)E;
  if (!chosen) up = 0.0f;
  const bool soft = a.scoring == MLXQ_ROUTE_SOFTMAX;
#pragma unroll
  for (int i = 0; i < NE; ++i) mine[i * 64 + lane] = z[i];
  __builtin_amdgcn_wave_barrier();
  const float zj = chosen ? mine[id] : -INFINITY;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < NE; ++i) mine[i * 64 + lane] = 0.0f;
  __builtin_amdgcn_wave_barrier();
  const auto larger = [](float u, float v) { return fmaxf(u, v); };  // of a number and NaN the number
  float top = -INFINITY;
  bool undefined = false;  // softmax of a row with NaN or +infinity
  // A token without an expert, as of a padded batch, passes nothing on, whatever its logits hold.
  const bool none = !__any(chosen);
  if (soft) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      top = fmaxf(top, z[i]);  // the last logit again past the end
      undefined |= !(z[i] < INFINITY);
    }
    top = lanes_reduce(top, larger);
    if (top == -INFINITY) top = 0.0f;
    undefined = __any(undefined);
  }
  float dot = 0.0f, dj;  // dj: dz of a chosen expert, or of a softmax without normalization d
  if (a.normalize) {
    const float most = lanes_reduce(zj, larger);
    float v, q = 1.0f;
    if (soft) {
      v = exp_of(zj - (top - most <= 745.13f ? most : top));
    } else {
      const float e = exp_of(-fabsf(zj)), big = 1.0f / (1.0f + e), small = e * big;
      q = zj >= 0.0f ? small : big;
      v = most < 0.0f && most >= -709.78f ? exp_of(zj - most) * q : zj >= 0.0f ? big : small;
    }
    if (!chosen) v = 0.0f;
    const float sum = wave_sum(v);
    v *= sum == 0.0f ? 0.0f : 1.0f / sum;
    dj = v * (up - wave_sum(up * v)) * q;
  } else if (soft) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      z[i] = i * 64 + lane < E ? exp_of(z[i] - top) : 0.0f;
      sum += z[i];
    }
    sum = wave_sum(sum);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < NE; ++i) z[i] *= inv;
    dot = wave_sum(chosen ? up * (exp_of(zj - top) * inv) : 0.0f);
    dj = up;
  } else {
    const float e = exp_of(-fabsf(zj)), big = 1.0f / (1.0f + e);
    dj = up * big * (e * big);
  }
  if (chosen) mine[id] = dj;
  __builtin_amdgcn_wave_barrier();
  T* out = dz + (int64_t)t * E;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = i * 64 + lane;
    const float v = mine[e];
    if (e < E) Act<T>::st(out, e, none ? 0.0f : undefined ? NAN : soft && !a.normalize ? z[i] * (v - dot) : v);
  }
}

// ---- the plan ------------------------------------------------------------------------------------

// Lanes of the wave whose expert is this lane's, as a mask: one ballot a bit.
__device__ __forceinline__ unsigned long long same_expert(int e, int bits) {
  unsigned long long m = ~0ull;
  for (int b = 0; b < bits; ++b) {
    const unsigned long long set = __ballot(e >> b & 1);
    m &= e >> b & 1 ? set : ~set;
  }
  return m;
}

// A run of choices, by one wave, 64 at a time and the loads of four times as many together: f(choice, whether there is
// one, its expert (E: none), lanes with the same one).
template <typename F>
__device__ __forceinline__ void walk(const int32_t* ids, int first, int last, int E, int bits, F&& f) {
  const int lane = threadIdx.x & 63;
  for (int c0 = first; c0 < last; c0 += 256) {
    int e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = ids[min(c0 + 64 * i + lane, last - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 64 * i + lane;
      if (c0 + 64 * i >= last) break;
      const int x = (unsigned)e[i] < (unsigned)E ? e[i] : E;
      f(c, c < last, x, same_expert(x, bits) & __ballot(c < last));
    }
  }
}

// Counts of each segment's experts, [segments][E + 1].  Sums of integers: the order of the additions does not matter.
__global__ __launch_bounds__(1024) void route_count_kernel(const int32_t* __restrict__ ids, int n, int E, int segment,
                                                           int32_t* __restrict__ counts) {
  __shared__ int count[1025];
  const int first = blockIdx.x * segment, last = min(n, first + segment);
  for (int e = threadIdx.x; e <= E; e += 1024) count[e] = 0;
  __syncthreads();
  for (int c = first + threadIdx.x; c < last; c += 1024) atomicAdd(&count[(unsigned)ids[c] < (unsigned)E ? ids[c] : E], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += 1024) counts[(int64_t)blockIdx.x * (E + 1) + e] = count[e];
}

// The plan of a few choices, by one workgroup: a part of them a wave.
__global__ __launch_bounds__(1024) void route_small_plan_kernel(const int32_t* __restrict__ ids, int n, int E, int bits,
                                                                int32_t* __restrict__ starts, int32_t* __restrict__ rows) {
  __shared__ int next[16][1025];  // a wave's counts, then where its next choice of an expert goes
  __shared__ int sums[1025 + 63];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, W = blockDim.x >> 6;
  const int per = ((n + W - 1) / W + 63) & ~63, first = min(n, w * per), last = min(n, first + per);
  for (int e = lane; e <= E; e += 64) next[w][e] = 0;
  __builtin_amdgcn_wave_barrier();
  walk(ids, first, last, E, bits, [&](int, bool live, int e, unsigned long long same) {
    if (live && lane == __builtin_ctzll(same)) next[w][e] += __popcll(same);
    __builtin_amdgcn_wave_barrier();
  });
  __syncthreads();
  for (int e = tid; e <= E; e += blockDim.x) {
    int s = 0;
    for (int k = 0; k < W; ++k) s += next[k][e];
    sums[e] = s;
  }
  __syncthreads();
  if (w == 0) {
    int before = 0;
    for (int e0 = 0; e0 <= E; e0 += 64) {
      const int e = e0 + lane, own = e <= E ? sums[e] : 0;
      int s = own;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d);
        if (lane >= d) s += o;
      }
      if (e <= E) {
        sums[e] = before + s - own;
        starts[e] = before + s - own;
      }
      before += __builtin_amdgcn_readlane(s, 63);
    }
  }
  __syncthreads();
  for (int e = tid; e <= E; e += blockDim.x) {
    int s = sums[e];
    for (int k = 0; k < W; ++k) {
      const int c = next[k][e];
      next[k][e] = s;
      s += c;
    }
  }
  __syncthreads();
  walk(ids, first, last, E, bits, [&](int c, bool live, int e, unsigned long long same) {
    const int at = live ? next[w][e] : 0, rank = __popcll(same & ((1ull << lane) - 1));
    __builtin_amdgcn_wave_barrier();
    if (live) {
      rows[at + rank] = c;
      if (rank == 0) next[w][e] = at + __popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  });
}

// Segment blockIdx.x's choices to their places: its experts' starts are the totals of all segments and the counts of earlier
// ones, of which each of sixteen waves adds up every sixteenth; within the segment each wave has a part, as in a small plan.
// 131048 choices of 256 experts: 22 us with four waves and a segment of 512 walked by one, 9 so.
constexpr int kPlaceWaves = 16;
__global__ __launch_bounds__(64 * kPlaceWaves) void route_place_kernel(const int32_t* __restrict__ ids, int n, int E, int bits, int segment,
                                                                       const int32_t* __restrict__ counts, int segments,
                                                                       int32_t* __restrict__ starts, int32_t* __restrict__ rows) {
  __shared__ int next[kPlaceWaves][1025];  // a wave's counts, then where its next choice of an expert goes
  __shared__ int sums[1025], base[1025], some[kPlaceWaves][2][64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, mine = blockIdx.x;
  for (int e0 = 0; e0 <= E; e0 += 64) {
    const int e = min(e0 + lane, E);
    int all = 0, before = 0;
#pragma unroll 8
    for (int s = w; s < segments; s += kPlaceWaves) {
      const int c = counts[(int64_t)s * (E + 1) + e];
      all += c;
      before += s < mine ? c : 0;
    }
    some[w][0][lane] = all;
    some[w][1][lane] = before;
    __syncthreads();
    if (w < 2 && e0 + lane <= E) {
      int s = 0;
#pragma unroll
      for (int k = 0; k < kPlaceWaves; ++k) s += some[k][w][lane];
      (w == 0 ? sums : base)[e] = s;
    }
    __syncthreads();
  }
  const int end = min(n, (mine + 1) * segment), per = ((end - mine * segment + kPlaceWaves - 1) / kPlaceWaves + 63) & ~63;
  const int first = min(end, mine * segment + w * per), last = min(end, first + per);
  for (int e = lane; e <= E; e += 64) next[w][e] = 0;
  __builtin_amdgcn_wave_barrier();
  walk(ids, first, last, E, bits, [&](int, bool live, int e, unsigned long long same) {
    if (live && lane == __builtin_ctzll(same)) next[w][e] += __popcll(same);
    __builtin_amdgcn_wave_barrier();
  });
  if (w == 0) {
    int before = 0;
    for (int e0 = 0; e0 <= E; e0 += 64) {
      const int e = e0 + lane, own = e <= E ? sums[e] : 0;
      int s = own;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d);
        if (lane >= d) s += o;
      }
      if (e <= E) {
        base[e] += before + s - own;
        if (mine == 0) starts[e] = before + s - own;
      }
      before += __builtin_amdgcn_readlane(s, 63);
    }
  }
  __syncthreads();
  for (int e = tid; e <= E; e += 64 * kPlaceWaves) {
    int s = base[e];
    for (int k = 0; k < kPlaceWaves; ++k) {
      const int c = next[k][e];
      next[k][e] = s;
      s += c;
    }
  }
  __syncthreads();
  walk(ids, first, last, E, bits, [&](int c, bool live, int e, unsigned long long same) {
    const int at = live ? next[w][e] : 0, rank = __popcll(same & ((1ull << lane) - 1));
    __builtin_amdgcn_wave_barrier();
    if (live) {
      rows[at + rank] = c;
      if (rank == 0) next[w][e] = at + __popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  });
}

constexpr int kOneGroup = 2048;  // choices that one workgroup sorts by itself
int64_t segment_of(int64_t n) { return ((n + 255) / 256 + 1023) / 1024 * 1024; }  // at most 256 segments

template <typename F>
int by_experts(int E, F&& f) {
  if (E <= 64) return f(std::integral_constant<int, 1>{});
  if (E <= 128) return f(std::integral_constant<int, 2>{});
  if (E <= 256) return f(std::integral_constant<int, 4>{});
  if (E <= 512) return f(std::integral_constant<int, 8>{});
  return f(std::integral_constant<int, 16>{});
}

// Four tokens a workgroup; those from the launch's first on.
template <typename T, typename F>
int by_tokens(const char* what, const RouteArgs& a, F&& launch) {
  return in_launches(what, ((int64_t)a.T + 3) / 4, 256, [&](int64_t group, unsigned grid) {
    const int64_t t = group * 4;
    RouteArgs part = a;
    part.logits = (const T*)a.logits + t * a.row_stride;
    part.T = (int)(a.T - t);
    part.ids += t * a.k;
    if (a.weights) part.weights += t * a.k;
    if (a.active) part.active += t;
    launch(part, t, grid);
  });
}

template <typename T>
int route(const RouteArgs& a, hipStream_t st) {
  return by_experts(a.E, [&](auto n) {
    constexpr int NE = decltype(n)::value;
    const bool wide = a.bias || (a.kept < a.groups && a.best > 1);
    return by_tokens<T>("route_experts", a, [&](const RouteArgs& part, int64_t, unsigned grid) {
      if (wide) route_kernel<T, NE, true><<<grid, 256, 0, st>>>(part);
      else route_kernel<T, NE, false><<<grid, 256, 0, st>>>(part);
    });
  });
}

template <typename T>
int route_backward(const RouteArgs& a, const float* dweights, void* dz, hipStream_t st) {
  return by_experts(a.E, [&](auto n) {
    return by_tokens<T>("route_experts_backward", a, [&](const RouteArgs& part, int64_t t, unsigned grid) {
      route_grad_kernel<T, decltype(n)::value><<<grid, 256, 0, st>>>(part, dweights + t * a.k, (T*)dz + t * a.E);
    });
  });
}

}  // namespace

int run_route(const RouteArgs& a, int dtype, hipStream_t st) {
  if (dtype == MLXQ_BFLOAT16) return route<uint16_t>(a, st);
  if (dtype == MLXQ_FLOAT16) return route<_Float16>(a, st);
  return route<float>(a, st);
}

int run_route_backward(const RouteArgs& a, int dtype, const float* dweights, void* dz, hipStream_t st) {
  if (dtype == MLXQ_BFLOAT16) return route_backward<uint16_t>(a, dweights, dz, st);
  if (dtype == MLXQ_FLOAT16) return route_backward<_Float16>(a, dweights, dz, st);
  return route_backward<float>(a, dweights, dz, st);
}

size_t route_plan_workspace(int64_t choices, int64_t E) {
  if (choices <= kOneGroup) return 0;
  const int64_t seg = segment_of(choices);
  return (size_t)((choices + seg - 1) / seg * (E + 1) * 4);
}

int run_route_plan(const int32_t* ids, int64_t choices, int64_t E, int32_t* starts, int32_t* rows, void* ws, hipStream_t st) {
  int bits = 0;
  while ((1 << bits) < E + 1) ++bits;
  if (choices <= kOneGroup) {
    const int waves = (int)std::min<int64_t>(16, std::max<int64_t>(1, (choices + 63) / 64));
    route_small_plan_kernel<<<1, 64 * waves, 0, st>>>(ids, (int)choices, (int)E, bits, starts, rows);
    return check_launch("route_plan");
  }
  const int64_t seg = segment_of(choices), n = (choices + seg - 1) / seg;
  route_count_kernel<<<(unsigned)n, 1024, 0, st>>>(ids, (int)choices, (int)E, (int)seg, (int32_t*)ws);
  if (int rc = check_launch("route_plan")) return rc;
  route_place_kernel<<<(unsigned)n, 64 * kPlaceWaves, 0, st>>>(ids, (int)choices, (int)E, bits, (int)seg, (const int32_t*)ws, (int)n, starts, rows);
  return check_launch("route_plan");
}

}  // namespace mlxq
