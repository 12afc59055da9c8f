// attention_stream.h — paged attention for few rows a key head (decode, drafted tokens) in any dtype,
// and for f32 at every size.
//
// Rows are (token, query head) pairs of one sequence and key head, so the heads that share a key head
// read it once.  A workgroup holds 16 * MT rows and a range of the sequence's keys; each of its waves
// walks its own units of keys (32 for 16-bit types, 16 for f32) with its own running maximum and sum
// (an online softmax), and the waves' results are joined in LDS at the end.  Long sequences are also
// split over workgroups, whose sums a second kernel joins.
//
// Scores are computed transposed, S^T = K Q^T, and so is the result, O^T = V^T P^T: the cache's layout
// is the A operand of both products, 16 bytes a lane and 1 KB a wave straight from memory, and a lane of S^T
// holds scores of one row.  With lane = 16 g + c, the D operand of the 16x16 products puts rows 4 g + i
// in lane (g, c): element i of tile t is key 16 t + 4 g + i.  f32 values arrive in that order.  16-bit values arrive
// as 8 keys a lane, group g = 2 b + a those from 8 a on of block b; two exchanges between lane groups
// (even_keys) turn two blocks into keys 4 g .. 4 g + 3 of either, the order of the weights.
//
// Bound by the cache's bytes for one token: no LDS and no barrier in the loop, and the next unit's keys
// are requested as soon as this one's are used.  Two sequences of up to 150001 tokens, 28 + 4 fp16 heads of 128: 62 us
// and 7 for the join, 307 MB at 5.0 TB/s (a plain read runs at 5.7-6.4).  48 of up to 6000, 64 + 8 heads of 64: 20 + 4 us;
// the workgroups of splits that short sequences lack take 2.5 ns each.  One of 777: 5 + 5 us, all latency.
// f32 prompts are bound by the f32 products, a sixteenth of bf16's rate: 3 prompts of up to 700 tokens over 900, 12
// heads of 80: 39 us, 57 TFLOP/s where a large f32 product reaches 153; their tiles fill the chip 1.5 times, half of
// them meet the diagonal or the shared part's end, and three waves a SIMD do not hide each other's chains of products,
// exchanges and exponentials (matrix cores 33 % busy; 2000 tokens at once, 8 heads of 64: 47 us, 88 TFLOP/s).
#pragma once

#include "paged.h"

namespace mlxq {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// acc += A (16 x one chunk a lane group) . B, one chunk = 8 16-bit or 4 f32 products deep a lane group.
template <typename T>
__device__ __forceinline__ f32x4 mma16(const u32x4& a, const u32x4& b, f32x4 acc) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), acc, 0, 0, 0);
    return acc;
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  }
}

// The four lane groups' values of a row: lanes c, 16 + c, 32 + c, 48 + c.
__device__ __forceinline__ float group_max(float v) {
  const uint32_t u = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float group_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A value that is infinite or NaN must not meet the weight 0 of a row that does not see it.  Where a unit of
// keys is hidden from some row, such values are taken out of the product (finite_mask) and, if there are any, added by a
// second product of codes with indicators of the rows' non-zero weights: +inf counts 1, -inf 128, NaN both,
// exact in all three types and, over at most 64 keys, in their sum.
//
// carries(): the sign bits of the result are those of the values (two to a word in 16-bit types) whose exponent bits
// are all set, where adding one at the exponent's lowest bit carries.
template <typename T>
constexpr uint32_t kCarry = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
template <typename T>
__device__ __forceinline__ uint32_t carries(uint32_t v) {
  constexpr uint32_t mask = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, _Float16) ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = sizeof(T) == 4 ? 0x00800000u : __is_same(T, _Float16) ? 0x04000400u : 0x00800080u;
  return (v & mask) + one;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_mask(uint32_t v) {
  const uint32_t t = carries<T>(v) & kCarry<T>;
  return sizeof(T) == 4 ? (t >> 31) - 1u : ~((t >> 15) * 0xffffu);
}
template <typename T>
__device__ __forceinline__ uint32_t value_code(uint32_t v) {
  constexpr uint32_t pos = sizeof(T) == 4 ? 0x3f800000u : __is_same(T, _Float16) ? 0x3c00u : 0x3f80u;  // 1
  constexpr uint32_t neg = sizeof(T) == 4 ? 0x43000000u : __is_same(T, _Float16) ? 0x5800u : 0x4300u;  // 128
  constexpr uint32_t both = sizeof(T) == 4 ? 0x43010000u : __is_same(T, _Float16) ? 0x5808u : 0x4301u; // 129
  const uint32_t bad = ~finite_mask<T>(v);
  if constexpr (sizeof(T) == 4) return bad & ((v & 0x007fffffu) ? both : v >> 31 ? neg : pos);
  constexpr uint32_t man = __is_same(T, _Float16) ? 0x03ffu : 0x007fu;
  const uint32_t lo = (v & man) ? both : (v & 0x8000u) ? neg : pos;
  const uint32_t hi = (v >> 16 & man) ? both : v >> 31 ? neg : pos;
  return bad & (lo | hi << 16);
}
template <typename T>
__device__ __forceinline__ uint32_t weight_code(uint32_t v) {
  if constexpr (sizeof(T) == 4) return v ? 0x3f800000u : 0u;
  constexpr uint32_t one = __is_same(T, _Float16) ? 0x3c00u : 0x3f80u;
  return (v & 0xffffu ? one : 0u) | (v >> 16 ? one << 16 : 0u);
}
__device__ __forceinline__ float decoded(float x) {
  const float n = floorf(x * (1.0f / 128.0f));
  return (x - 128.0f * n > 0.0f ? INFINITY : 0.0f) + (n > 0.0f ? -INFINITY : 0.0f);
}
template <typename T>
__device__ __forceinline__ u32x4 each(u32x4 v, uint32_t (*f)(uint32_t)) {
  return u32x4{f(v[0]), f(v[1]), f(v[2]), f(v[3])};
}

// The sum of a pair of 16-bit weights, added to acc.
template <typename T>
__device__ __forceinline__ float pair_sum(uint32_t v, float acc) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  if constexpr (__is_same(T, _Float16))
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, v), f16x2{(_Float16)1.0f, (_Float16)1.0f}, acc, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, acc, false);
}

// The running maximum a row's exponents are taken against moves only when a score passes it by this many
// units of log 2: weights up to 2^8 are as exact as weights up to 1 (fp16's end at 2^16), and the sums
// are rescaled rarely.
constexpr float kSlack = 8.0f;

// Whether any wave of the workgroup says so.  flags: LDS, one for each of the NW waves, used for nothing else.
template <int NW>
__device__ __forceinline__ bool any_wave(bool v, int* flags) {
  if ((threadIdx.x & 63) == 0) flags[threadIdx.x >> 6] = v;
  __syncthreads();
  int r = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) r |= flags[i];
  return __builtin_amdgcn_readfirstlane(r) != 0;
}

// Rows (keys [lo, lo + span)) that see a key of [from, to) whose table entry names no page get a NaN sum.
template <int N>
__device__ __forceinline__ void poison(const Batch& bt, const int32_t* table, int from, int to, const int (&lo)[N],
                                       const int (&span)[N], float (&sum)[N]) {
  for (int i = from >> bt.page_log2; i <= (to - 1) >> bt.page_log2; ++i) {
    if ((unsigned)table[i] < (unsigned)bt.pages) continue;
    const int f = max(i << bt.page_log2, from), t = min((i + 1) << bt.page_log2, to);
#pragma unroll
    for (int m = 0; m < N; ++m)
      if (max(f, lo[m]) < min(t, lo[m] + span[m])) sum[m] = __builtin_nanf("");
  }
}

constexpr float kLog2e = 1.44269504088896341f;

// What happens to a score before the softmax: nothing, a cap, or a bias by distance (capped before it if
// softcap is set).  kFar: a cap past kNearCap, in 16-bit types, and then the bias if there is one.
enum Bend : int { kPlain = 0, kCap = 1, kBias = 2, kFar = 3 };
constexpr float kNearCap = 256.0f;
// A capped or biased score, in units of log 2, from q.k and the distance of key and row.  With x = score / cap, cap tanh(x) is
// cap - 2 cap / (exp(2 x) + 1), in 16-bit types with the hardware's exponential and reciprocal, off by up to 5 2^-24 cap: up to
// kNearCap less than a third of what rounding a weight to fp16 is.  Past it, where |x| < 1/4, it is the first four terms of
// tanh's series times the cap, score (1 - x^2/3 + 2 x^4/15 - 17 x^6/315), off by 6 2^-24 of the score, whatever the
// cap.  As kernels of its own, since both in one take registers from the nearer caps.
// AttnArgs::scale is 2 scale / (cap ln 2) with a cap, so that z is 2 x in units of log 2, and scale / ln 2 without, as
// score_scale always is; cap2 is softcap / ln 2.
template <typename T, int BEND>
__device__ __forceinline__ float bent_score(const AttnArgs& a, float qk, float slope2, float distance) {
  constexpr float kHalf = 0.34657359027997265f;  // ln 2 / 2: x = kHalf z
  float z = qk * a.scale;
  if (BEND == kCap || BEND == kFar || a.softcap > 0.0f) {
    if constexpr (sizeof(T) == 4) {
      z = a.cap2 * tanhf(z * kHalf);
    } else {
      const float bent = fmaf(-2.0f * a.cap2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(z) + 1.0f), a.cap2);
      if constexpr (BEND == kFar) {
        constexpr float h2 = kHalf * kHalf, c1 = -h2 / 3.0f, c2 = 2.0f * h2 * h2 / 15.0f, c3 = -17.0f * h2 * h2 * h2 / 315.0f;
        const float score = qk * a.score_scale, t = z * z, series = fmaf(score * t, fmaf(t, fmaf(t, c3, c2), c1), score);
        z = fabsf(z) < 0.25f / kHalf ? series : bent;
      } else {
        z = bent;
      }
    }
  }
  if constexpr (BEND == kBias || BEND == kFar) z = fmaf(-slope2, fabsf(distance), z);
  return z;
}
template <int BEND>
__device__ __forceinline__ float slope_of(const AttnArgs& a, int qh) {
  return BEND == kBias || (BEND == kFar && a.slopes) ? a.slopes[qh] * kLog2e : 0.0f;
}

// What a row sees of the tokens that have a page.
struct RowRange {
  int lo, hi;
};
__device__ __forceinline__ RowRange row_range(const AttnArgs& a, const Seq& s, int p, int prefix) {
  const int hi = a.causal ? min(s.paged, max(p + 1, prefix)) : s.paged;
  return {a.window ? max(0, p + 1 - a.window) : 0, hi};
}
// Where the sum of weights of the row at place p starts: at NaN, which stays, if the row sees a token past the table.
__device__ __forceinline__ float first_sum(const AttnArgs& a, const Seq& s, int p, int prefix) {
  if (s.L == s.paged) return 0.0f;
  return !a.causal || max(p + 1, prefix) > s.paged ? __builtin_nanf("") : 0.0f;
}

// First to last key that any row of [row0, row1] sees, those that every one sees, and this split's.
struct KeyRange {
  int lo, hi;          // any row
  int lo_all, hi_all;  // every row
};
__device__ __forceinline__ KeyRange key_range(const AttnArgs& a, const Seq& s, int row0, int row1, int prefix) {
  const RowRange f = row_range(a, s, s.L - s.n + a.by_g.div(row0), prefix), l = row_range(a, s, s.L - s.n + a.by_g.div(row1), prefix);
  return {f.lo, l.hi, l.lo, f.hi};
}

// v: a lane group's 8 keys of a block, see above, becomes 4 keys of block 0 and 4 of block 1.  With x and y the
// halves of v by lane group, x = (x0, x1, x2, x3): rows 1 and 3 of x change places with rows 0 and 2 of y, then the upper
// half of x with the lower half of y, which leaves x = (x0, y0, x1, y1) and y = (x2, y2, x3, y3).
__device__ __forceinline__ u32x4 even_keys(u32x4 v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    auto a = __builtin_amdgcn_permlane16_swap(v[i], v[2 + i], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(a[0], a[1], false, false);
    v[i] = b[0];
    v[2 + i] = b[1];
  }
  return v;
}

// Waves a SIMD for DT * MT = d: as many as the registers hold without spilling, and one step more in two places that are
// faster with spills (16-bit types; narrower heads, caps and biases spill more than full heads).  Two row tiles of 128
// features, 12 to 66 registers: 8 sequences of 4 tokens over 4000, 32 + 4 heads, bf16 23.4 us, fp16 24.1, one wave a SIMD
// 28.6 and 28.9, and 19 to 37 % more with a cap, a bias or heads of 112.  One of 64 features at four waves, 0 to 28
// registers: 49 sequences of 300 to 6000 tokens, 64 + 8 heads, bf16 34.8 us, fp16 35.7, three waves 37.8 and 38.5; 8 of
// 5000 and 32 of 777 tokens within 6 % either way.
template <typename T>
constexpr int stream_waves(int d, int mt = 1) {
  if (sizeof(T) == 4) return d <= 80 ? 3 : d <= 128 ? 2 : 1;
  return d <= 64 ? 4 : d <= 128 || mt == 2 ? 2 : 1;
}

// Kernels of one wave a SIMD keep queries and results in the accumulation registers, which matrix products read and write
// directly: held there wherever anything else uses them, since the compiler, left to itself, moves all results out and
// back every unit or tile.
template <bool ACC, typename V>
__device__ __forceinline__ void pin(V& v) {
  if constexpr (ACC) asm volatile("" : "+a"(v));
}

// FULL: head_dim is DT, else below it and the rest of DT is zeros.
template <typename T, int DT, int MT, int BEND, bool FULL>
__global__ __launch_bounds__(256, stream_waves<T>(DT * MT, MT)) void attn_stream_kernel(AttnArgs a) {
  constexpr int C = Elem<T>::C, KU = 4 * C, NT = KU / 16, NS = DT / (4 * C), ND = DT / 16, TM = 16 * MT, NW = 4;
  constexpr bool ACC = stream_waves<T>(DT * MT, MT) == 1;
  constexpr int JD = DT * MT < 256 ? DT : DT / 2;  // features joined at a time: all that 64 KB hold
  __shared__ float lm[NW][TM], ll[NW][TM];
  __shared__ int flags[NW];
  __shared__ __align__(16) float lo_[NW][TM][JD + 4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  // Workgroups go round the chip's eight dies in order of their number: the (tile, head) items of a split come
  // together, each split's turned by one, so that a long sequence's splits fall on all dies.
  const int z = a.by_items.div(blockIdx.x), turn = blockIdx.x - z * a.items + (z - a.by_items.div(z) * a.items);
  const int item = turn < a.items ? turn : turn - a.items, unit = a.by_hkv.div(item), h = item - unit * a.Hkv;
  const Batch& bt = a.batch;
  const int D = FULL ? DT : a.D;
  const int blog = bt.page_log2 - 4, bmask = (1 << blog) - 1, cu = a.chunk / KU;  // blocks of a page, units of a split
  auto tiles_of = [&](const Seq& s) { return (s.n * a.G + TM - 1) / TM; };
  int b = unit, first = 0;
  if (!a.direct && !Finder(bt, tiles_of).find(unit, b, first)) return;
  const Seq s = load_seq(bt, b);
  const int rows = s.n * a.G, prefix = a.prefix ? a.prefix[b] : 0;
  const int last = a.direct ? tiles_of(s) : first + 1;
  const int32_t* table = bt.tables + b * bt.table_stride;
  const int64_t head = ((int64_t)h << bt.page_log2) * D;
  const T *kp = (const T*)a.k + head, *vp = (const T*)a.v + head;

  for (int at = first; at < last; ++at) {
    const int tile = a.direct ? at : tiles_of(s) - 1 - at;  // the longest first
    const int row0 = tile * TM, row1 = min(rows, row0 + TM) - 1;
    const KeyRange kr = key_range(a, s, row0, row1, prefix);
    const int ub = kr.lo / KU, ue = kr.hi > kr.lo ? (kr.hi + KU - 1) / KU : ub;
    const int ns = max(1, min(a.S, a.by_chunk.div((ue - ub) * KU + a.chunk - 1)));
    if (z >= ns) continue;
    const int u0 = ub + z * cu, u1 = z == a.S - 1 ? ue : min(ue, u0 + cu);
    const int blo = kr.lo >> 4, bhi = (kr.hi - 1) >> 4;  // blocks with keys that are seen

    // A unit's blocks of 16 keys: their pages, and the blocks' first elements.  Blocks that no row sees are
    // never looked up: their entries may name nothing.
    bool bad = false;
    auto page_of = [&](int blk) { return table[min(max(blk, blo), bhi) >> blog]; };
    auto block_at = [&](int blk, int page, int64_t stride) {
      const bool in = (unsigned)page < (unsigned)bt.pages;
      bad |= !in;
      return (int64_t)(in ? page : 0) * stride + (int64_t)(min(max(blk, blo), bhi) & bmask) * 16 * D;
    };
    u32x4 kf[NT][NS], vf[ND];
    auto load_k = [&](int u, int pg0, int pg1) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const T* at = kp + block_at(u * NT + t, t ? pg1 : pg0, a.k_page) + lane * C;
#pragma unroll
        for (int k = 0; k < NS; ++k)
          kf[t][k] = FULL || (4 * k + g) * C < D ? load_chunk(at + 64 * k * C) : u32x4{0, 0, 0, 0};
      }
    };
    auto load_v = [&](int u, int pg0, int pg1) {
      const T* base = vp + block_at(u * (KU / 16), pg0, a.v_page);
      if constexpr (KU == 32) {
        const T* other = vp + block_at(u * 2 + 1, pg1, a.v_page);
        base = g >= 2 ? other : base;
      }
      const T* at = base + ((KU == 32 ? g & 1 : g) * D + c) * C;
#pragma unroll
      for (int d = 0; d < ND; ++d) vf[d] = FULL || 16 * d < D ? load_chunk(at + 16 * d * C) : u32x4{0, 0, 0, 0};
    };
    int u = u0 + w, pg0 = 0, pg1 = 0;
    if (u < u1) {
      pg0 = page_of(u * (KU / 16));
      pg1 = KU == 32 ? page_of(u * 2 + 1) : pg0;
      load_k(u, pg0, pg1);
      load_v(u, pg0, pg1);
    }

    // This lane's rows.
    int place[MT], lo[MT], span[MT];
    float slope[MT];
    u32x4 qf[MT][NS];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = min(row0 + m * 16 + c, row1), i = a.by_g.div(r), qh = h * a.G + (r - i * a.G);
      const int p = s.L - s.n + i;
      const RowRange rr = row_range(a, s, p, prefix);
      place[m] = p;
      lo[m] = rr.lo;
      span[m] = max(rr.hi - rr.lo, 0);
      slope[m] = slope_of<BEND>(a, qh);
      const T* q = (const T*)a.q.p + (s.q0 + i) * a.q.ts + qh * a.q.hs;
#pragma unroll
      for (int k = 0; k < NS; ++k) qf[m][k] = FULL || (4 * k + g) * C < D ? load_chunk(q + (4 * k + g) * C) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < NS; ++k) pin<ACC>(qf[m][k]);
    }
    f32x4 o[MT][ND];
    float ref[MT], sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      ref[m] = -INFINITY;
      sum[m] = first_sum(a, s, place[m], prefix);
#pragma unroll
      for (int d = 0; d < ND; ++d) o[m][d] = f32x4{0, 0, 0, 0};
    }
    const float cs = BEND != kPlain ? 1.0f : a.scale;

    for (; u < u1; u += NW) {
      const bool more = u + NW < u1;
      if (more) {
        pg0 = page_of((u + NW) * (KU / 16));
        pg1 = KU == 32 ? page_of((u + NW) * 2 + 1) : pg0;
      }
      f32x4 st[MT][NT];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          st[m][t] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < NS; ++k)
            if (FULL || 4 * k * C < D) st[m][t] = mma16<T>(kf[t][k], qf[m][k], st[m][t]);
        }
      if (more) load_k(u + NW, pg0, pg1);
      const int key0 = u * KU + 4 * g;
      const bool part = u * KU < kr.lo_all || (u + 1) * KU > kr.hi_all;
      if (BEND != kPlain || part) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = key0 + 16 * t + i;
              float v = st[m][t][i];
              if constexpr (BEND != kPlain) v = bent_score<T, BEND>(a, v, slope[m], (float)(j - place[m]));
              if (part) v = (unsigned)(j - lo[m]) < (unsigned)span[m] ? v : -INFINITY;
              st[m][t][i] = v;
            }
      }
      u32x4 pf[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float v = st[m][0][0];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) v = fmaxf(v, st[m][t][i]);
        v = group_max(v) * cs;
        const bool up = v > ref[m] + kSlack;
        if (__any(up)) {
          const float now = up ? v : ref[m];
          const float alpha = up ? __builtin_amdgcn_exp2f(ref[m] - now) : 1.0f;
          ref[m] = now;
          sum[m] *= alpha;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            pin<ACC>(o[m][d]);
            o[m][d] *= alpha;
            pin<ACC>(o[m][d]);
          }
        }
        const float neg = ref[m] == -INFINITY ? 0.0f : -ref[m];  // nothing seen yet: all weights are exp2(-inf)
        float e[C], add = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          e[i] = __builtin_amdgcn_exp2f(fmaf(st[m][i / 4][i % 4], cs, neg));
          add += e[i];
        }
        sum[m] += add;
        // 16-bit types: the softmax weights are rounded to the type for the product with the values (their
        // f32 sum is not): half a unit in the last place of each weight, as the values themselves carry.
        pf[m] = pack_chunk<T>(e);
      }
      if constexpr (KU == 32) {
#pragma unroll
        for (int d = 0; d < ND; ++d) vf[d] = even_keys(vf[d]);
      }
      if (part) {
        uint32_t nf = 0;
#pragma unroll
        for (int d = 0; d < ND; ++d) nf |= carries<T>(vf[d][0]) | carries<T>(vf[d][1]) | carries<T>(vf[d][2]) | carries<T>(vf[d][3]);
        if (__builtin_expect(__any((nf & kCarry<T>) != 0), 0)) {
#pragma unroll
          for (int d = 0; d < ND; ++d) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const f32x4 x = mma16<T>(each<T>(vf[d], value_code<T>), each<T>(pf[m], weight_code<T>), f32x4{0, 0, 0, 0});
              pin<ACC>(o[m][d]);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[m][d][i] += decoded(x[i]);
              pin<ACC>(o[m][d]);
            }
            vf[d] &= each<T>(vf[d], finite_mask<T>);
          }
        }
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (FULL || 16 * d < D) o[m][d] = mma16<T>(vf[d], pf[m], o[m][d]);
      if (more) load_v(u + NW, pg0, pg1);
    }

    // Join the waves: maxima and sums first, then the results.
    if (any_wave<NW>(bad, flags)) poison(bt, table, max(u0 * KU, kr.lo), min(u1 * KU, kr.hi), lo, span, sum);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float t = group_sum(sum[m]);
      if (g == 0) {
        lm[w][m * 16 + c] = ref[m];
        ll[w][m * 16 + c] = t;
      }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < NW; ++i) top = fmaxf(top, lm[i][m * 16 + c]);
      const float f = __builtin_amdgcn_exp2f(ref[m] - (top == -INFINITY ? 0.0f : top));
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        pin<ACC>(o[m][d]);
        o[m][d] *= f;
      }
    }
#pragma unroll
    for (int j0 = 0; j0 < DT; j0 += JD) {
      if (j0) __syncthreads();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int d = 0; d < JD / 16; ++d) *reinterpret_cast<f32x4*>(&lo_[w][m * 16 + c][16 * d + 4 * g]) = o[m][j0 / 16 + d];
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < TM * (JD / 4); i += 64 * NW) {
        const int rr = i / (JD / 4), dj = (i - rr * (JD / 4)) * 4, d = j0 + dj, r = row0 + rr;
        if (r > row1 || d >= D) continue;
        f32x4 v = {0, 0, 0, 0};
        float top = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          v += *reinterpret_cast<const f32x4*>(&lo_[k][rr][dj]);
          top = fmaxf(top, lm[k][rr]);
        }
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < NW; ++k) l += ll[k][rr] * __builtin_amdgcn_exp2f(lm[k][rr] - base);
        const int tok = a.by_g.div(r), qh = h * a.G + (r - tok * a.G);
        const int64_t orow = (int64_t)(s.q0 + tok) * a.Hkv * a.G + qh;
        if (a.S > 1 && z == 0 && d == 0) a.splits[orow] = ns;
        if (ns > 1) {
          *reinterpret_cast<f32x4*>(a.part + (orow * a.S + z) * D + d) = v;
          if (d == 0) *reinterpret_cast<f32x2*>(a.ml + (orow * a.S + z) * 2) = f32x2{top, l};
        } else {
          if (a.sinks) l += __builtin_amdgcn_exp2f(a.sinks[qh] * kLog2e - base);
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          T* y = (T*)a.out.p + (s.q0 + tok) * a.out.ts + qh * a.out.hs + d;
          if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(y) = v * inv;
          else *reinterpret_cast<u32x2*>(y) = u32x2{Elem<T>::pack2(v[0] * inv, v[1] * inv), Elem<T>::pack2(v[2] * inv, v[3] * inv)};
        }
      }
    }
    if (at + 1 < last) __syncthreads();
  }
}

template <typename T, int DT, int MT, bool FULL>
static int launch_stream_of(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
  const dim3 grid((unsigned)plan.blocks);
  if constexpr (sizeof(T) == 2) {
    if (a.softcap > kNearCap) {
      hipLaunchKernelGGL((attn_stream_kernel<T, DT, MT, kFar, FULL>), grid, dim3(256), 0, st, a);
      return check_launch("paged_attention");
    }
  }
  if (a.slopes) hipLaunchKernelGGL((attn_stream_kernel<T, DT, MT, kBias, FULL>), grid, dim3(256), 0, st, a);
  else if (a.softcap > 0.0f) hipLaunchKernelGGL((attn_stream_kernel<T, DT, MT, kCap, FULL>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((attn_stream_kernel<T, DT, MT, kPlain, FULL>), grid, dim3(256), 0, st, a);
  return check_launch("paged_attention");
}
template <typename T, int DT, int MT>
static int launch_stream(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
  return a.D == DT ? launch_stream_of<T, DT, MT, true>(a, plan, st) : launch_stream_of<T, DT, MT, false>(a, plan, st);
}

// The narrowest width that holds the heads: what is past them costs registers, and with them waves a SIMD (f32, 400
// tokens over 700, 4 heads: 80 wide 21.5 us as 80 and 28.9 as 128, 96 wide 24.9 and 32.1; bf16, 32 single tokens over up to
// 4000, 8 heads of 96: 78 and 84).
template <typename T>
static int stream_of(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
  if (plan.rows == 16) {
    if (a.D <= 64) return launch_stream<T, 64, 1>(a, plan, st);
    if constexpr (sizeof(T) == 4)
      if (a.D <= 80) return launch_stream<T, 80, 1>(a, plan, st);
    if (a.D <= 96) return launch_stream<T, 96, 1>(a, plan, st);
    if (a.D <= 128) return launch_stream<T, 128, 1>(a, plan, st);
    return launch_stream<T, 256, 1>(a, plan, st);
  }
  if constexpr (sizeof(T) == 2) {
    if (a.D <= 64) return launch_stream<T, 64, 2>(a, plan, st);
    if (a.D <= 96) return launch_stream<T, 96, 2>(a, plan, st);
    return launch_stream<T, 128, 2>(a, plan, st);
  }
  return set_error(MLXQ_EINVAL, "paged_attention: no kernel for %d rows", plan.rows);
}

}  // namespace mlxq
