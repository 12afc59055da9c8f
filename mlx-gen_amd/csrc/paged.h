// paged.h — the paged-cache operators: device helpers shared by their kernels, and the launches the
// ABI layer calls.  The cache's layout is described in include/mlxq.h.
#pragma once

#include "mlxq_common.h"

namespace mlxq {

// The elements of one dtype: a chunk is 16 bytes, the unit of every load.
template <typename T>
struct Elem;  // T: uint16_t (bf16 bits), _Float16, float
template <>
struct Elem<uint16_t> {
  static constexpr int C = 8;
  static __device__ __forceinline__ float get(const u32x4& v, int e) {
    return e & 1 ? __uint_as_float(v[e >> 1] & 0xffff0000u) : __uint_as_float(v[e >> 1] << 16);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) { return pack_bf16x2(a, b); }
};
template <>
struct Elem<_Float16> {
  static constexpr int C = 8;
  static __device__ __forceinline__ float get(const u32x4& v, int e) { return e & 1 ? f16_hi(v[e >> 1]) : f16_lo(v[e >> 1]); }
  // Round to nearest even; v_cvt_pkrtz would truncate.
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
  }
};
template <>
struct Elem<float> {
  static constexpr int C = 4;
  static __device__ __forceinline__ float get(const u32x4& v, int e) { return __uint_as_float(v[e]); }
};

// C floats to a chunk.
template <typename T>
__device__ __forceinline__ u32x4 pack_chunk(const float* f) {
  u32x4 o;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = Elem<T>::pack2(f[2 * i], f[2 * i + 1]);
  }
  return o;
}

template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* p) {
  return *reinterpret_cast<const u32x4*>(p);
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const u32x4& v) {
  *reinterpret_cast<u32x4*>(p) = v;
}

// n / d for 0 <= n < 2^31 by a product: m = ceil(2^(31 + l) / d) with l = ceil(log2 d) is off from 2^(31 + l) / d by less
// than 1, so n m 2^-(31 + l) by less than 2^-l <= 1 / d.  A division by a runtime value is some twenty instructions,
// and a short launch's time is, for a good part, the fetching of its instructions.
struct Divisor {
  uint32_t d = 1, mul = 0, shift = 0;
  Divisor() = default;
  explicit Divisor(int64_t div) : d((uint32_t)div) {
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    if (l == 0) return;
    mul = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
    shift = l - 1;
  }
  __device__ __forceinline__ int div(int n) const { return mul ? (int)(__umulhi((uint32_t)n, mul) >> shift) : n; }
};

// [token][head][feature] view; strides in elements.
struct Heads {
  const void* p;
  int64_t ts, hs;
};

// A step's sequences (mlxq_paged_batch), with what every kernel checks them against.
struct Batch {
  const int32_t* tables;
  const int32_t* q_starts;
  const int32_t* kv_lens;
  int64_t table_stride;
  int B, T;
  int capacity;   // tokens that the table's width names, a multiple of 16 below 2^30; those past it have no page
  int page_log2;  // log2(page_size)
  int pages;
};

// One sequence: its new tokens are [q0, q0 + n) of the step and places [L - n, L) of the sequence, of which those below
// `paged` have a page.
struct Seq {
  int q0, n, L, paged;
};

__device__ __forceinline__ Seq load_seq(const Batch& a, int b) {
  int s = a.q_starts[b], e = a.q_starts[b + 1], L = a.kv_lens[b];
  s = min(max(s, 0), a.T);
  e = min(max(e, s), a.T);
  L = min(max(L, 0), 0x7fffffe0);  // a place and the end of its block fit 31 bits
  return {s, e - s, L, min(L, a.capacity)};
}

// Sequences cut into units (blocks of tokens, tiles of rows, ranges of keys): finds the sequence of a unit and the
// unit's place in it.  Every wave runs it by itself, 64 sequences at a time: a lane counts the units of one, an
// inclusive scan adds them up.  Units are asked for in ascending order, and the scan goes on from where it is.
template <typename F>
struct Finder {
  const Batch& a;
  F count;  // Seq -> its units
  int base = 0, before = 0, n = 0, sum = 0;

  __device__ __forceinline__ Finder(const Batch& batch, F f) : a(batch), count(f) { scan(); }
  __device__ __forceinline__ void scan() {
    const int lane = threadIdx.x & 63, i = base + lane;
    n = i < a.B ? count(load_seq(a, i)) : 0;
    sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int t = __shfl_up(sum, d);
      if (lane >= d) sum += t;
    }
  }
  // False when there is no unit u.
  __device__ __forceinline__ bool find(int u, int& b, int& at) {
    while (true) {
      const unsigned long long past = __ballot(sum > u - before);
      if (past) {
        const int l = __builtin_ctzll(past);
        b = base + l;
        at = u - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l));
        return true;
      }
      if (base + 64 >= a.B) return false;
      before += __builtin_amdgcn_readlane(sum, 63);
      base += 64;
      scan();
    }
  }
};
template <typename F>
Finder(const Batch&, F) -> Finder<F>;

struct RotaryArgs {
  const float* table;        // [rows, R/2, 2]; null: no rotation
  const int32_t* positions;  // [T] or null (cache_append: the token's place)
  int rows, R, interleaved, inverse;
};

struct AppendArgs {
  Heads k, v, q, q_out;  // q.p null: no queries
  void *k_cache, *v_cache;
  int64_t k_page, v_page;  // elements between pages
  Batch batch;
  RotaryArgs rot;
  int Hkv, Hq, D;
  int direct;  // unit u is the u-th sequence (each loops over its blocks); 0: by Finder
};

struct AttnArgs {
  Heads q, out;
  const void *k, *v;
  int64_t k_page, v_page;
  Batch batch;
  int Hkv, G, D;
  Divisor by_hkv, by_g, by_items;  // by_items: (tile, head) pairs of the streaming kernel's grid
  int items;
  int S, chunk;       // splits of a sequence's tokens, tokens in each (a multiple of 128, tiled of 64; the last takes the rest)
  Divisor by_chunk;
  float scale;          // multiplies q.k into units of log 2 (with a cap: see bent_score)
  float softcap, cap2, score_scale;  // softcap 0: none; see bent_score
  int causal, window, direct;  // direct: item u is the u-th sequence, else by Finder
  const int32_t* prefix;
  const float *slopes, *sinks;
  float* part;  // [T * Hq, S, D] sums of each split, then their (maximum, sum) pairs and the counts of
  float* ml;    // [T * Hq, S, 2]
  int* splits;  // [T * Hq]; null when S is 1
};

int run_rotary(const Heads& x, int dtype, int64_t T, int64_t H, int64_t D, const RotaryArgs& r, const Heads& y,
               hipStream_t st);
int run_rotary_table(const double* inv_freq, int64_t half, double magnitude, int64_t positions, float* table,
                     hipStream_t st);
int run_cache_append(const AppendArgs& a, int dtype, int64_t units, hipStream_t st);
int run_copy_pages(void* cache, int64_t planes, int64_t plane_stride, int64_t pages, int64_t page_bytes,
                   int64_t page_stride, const int32_t* src, const int32_t* dst, int64_t count, int32_t* tables,
                   int64_t rows, int64_t width, int64_t table_stride, hipStream_t st);

constexpr int kMaxSplits = 256;  // the join gives each a thread

// How an attention call is cut up: rows of a workgroup's tile, splits of the tokens, and the grid.
struct AttnPlan {
  int rows = 16, S = 1, chunk = 0;
  bool tiled = false, direct = false;
  int64_t blocks = 0;  // workgroups (tiled: times S)
  size_t ml = 0, splits = 0, total = 0;  // workspace: byte offsets of ml and splits, and its size
};
AttnPlan plan_attention(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int dtype, int64_t B, int64_t max_q,
                        int64_t max_kv, int64_t window, bool causal);
int run_attention(const AttnArgs& a, int dtype, const AttnPlan& plan, hipStream_t st);
// The instances of the streaming kernel, by dtype.
int run_attn_stream_bf16(const AttnArgs& a, const AttnPlan& plan, hipStream_t st);
int run_attn_stream_f16(const AttnArgs& a, const AttnPlan& plan, hipStream_t st);
int run_attn_stream_f32(const AttnArgs& a, const AttnPlan& plan, hipStream_t st);
// The instances of the tiled kernel.
int run_attn_tile_bf16(const AttnArgs& a, const AttnPlan& plan, hipStream_t st);
int run_attn_tile_f16(const AttnArgs& a, const AttnPlan& plan, hipStream_t st);

}  // namespace mlxq
